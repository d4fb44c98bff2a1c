// Orthogonalisation of matrices by Newton-Schulz products, for optimizers that step along the orthogonal factor of an update.
//
//   X = G / (|G|_F + eps); `steps` times: A = X X^T (X^T X for a matrix of more rows than columns), P = b A + c A^2, X <- a X + P X
//   (X P): an odd polynomial of degree five applied to the singular values.
//
// Arithmetic. Operands of the products are FP16 (11 bits, as many as TF32 has, at twice its rate; 8 bits of BF16 would be 5 % off for
// matrices with a few strong directions), sums FP32. The iterate is carried as the sum of two FP16 numbers, X = hi + lo: the product
// takes hi, the linear term a X takes both. With hi alone the rounding of the strong directions, spread over all directions and
// amplified a-fold per step as the weak ones are, is 0.8 % of the result for strong directions 20 times the others (3 % for 200
// times), with the pair 0.02-0.2 %. For small matrices, and for all where the caller asks for it, A, P and the operand X are pairs too. X is
// kept times 2^10, which takes its elements (about 1 / sqrt(rows * cols)) out of the range where FP16 loses bits.
//
// Large matrices: four 5632 x 2048 take 1.72 ms for five steps (925 TFLOP/s; 1.45 to 1.5 ms of pure noise). By themselves A has the
// tensor pipe at work 72 % of its cycles, X 74 %, P, with two rounds of short tiles, 51 %. Small ones wait for the chain of three products a
// step (three 512 x 512: 87 us, 5.2 a launch), the smallest for the exchanges of a cluster (128 x 1000: 67 us).
#include "common.cuh"
#include "tcgen05.cuh"

#include <algorithm>

namespace {
using namespace gdb_t5;

constexpr float NS_UP = 1024.0f, NS_DOWN = 1.0f / 1024.0f;
constexpr int NS_NORM_BLOCKS = 256;   // partial sums of a matrix's squares, at most

// ------------------------------------------------------------------ |G|_F and the first iterate
// eight consecutive elements of a row, zeros behind its end
template <typename T>
__device__ __forceinline__ void ns_load8(const T *p, unsigned left, bool vec, float (&f)[8])
{
    if (vec) {
        if constexpr (sizeof(T) == 2) {
            gdb_vec8<T> v;
            v.raw = __ldg(reinterpret_cast<const uint4 *>(p));
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = v.get(e);
        } else {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
            f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (unsigned)e < left ? gdb_io<T>::ld(p, e) : 0.0f;
    }
}
// Sums of squares are FP64, so that neither 1e38 nor 1e-38 leaves the range; eight squares are added in FP32 first where that holds them
// (one conversion in place of eight: four 5632 x 2048 BF16 matrices 60 -> 25 us).
__device__ __forceinline__ double ns_squares(const float (&f)[8])
{
    float most = 0.0f, s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        most = fmaxf(most, fabsf(f[e]));
        s = fmaf(f[e], f[e], s);
    }
    if (most == 0.0f || (most > 1.0e-12f && most < 1.0e18f)) return (double)s;   // (NaN among the elements: in s)
    double t = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) t += (double)f[e] * (double)f[e];
    return t;
}
__device__ __forceinline__ float2 ns_two(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
// f times the factor as the sum of two FP16 numbers
__device__ __forceinline__ void ns_halves(const float (&f)[8], double factor, float ff, uint4 &hi, uint4 &lo)
{
    const bool normal = ff < 3.0e38f && ff > 1.2e-38f;   // ff, the factor in FP32, is a normal number
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float u = normal ? f[2 * e] * ff : (float)((double)f[2 * e] * factor), v = normal ? f[2 * e + 1] * ff : (float)((double)f[2 * e + 1] * factor);
        const uint32_t p = half_pack<__half>::pack(u, v);
        const float2 r = ns_two(p);
        (&hi.x)[e] = p;
        (&lo.x)[e] = half_pack<__half>::pack(u - r.x, v - r.y);
    }
}
// The matrix is taken as one row of `count` elements.
template <typename T>
__global__ void __launch_bounds__(256)
ns_norm_kernel(const T *__restrict__ g, double *__restrict__ partial, size_t count, bool vec)
{
    gdb_pdl_sync();
    __shared__ double sh[8];
    const T *m = g + (size_t)blockIdx.y * count;
    double t = 0.0;
    const size_t stride = (size_t)gridDim.x * blockDim.x * 8U;
#pragma unroll 4
    for (size_t i = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 8U; i < count; i += stride) {
        float f[8];
        ns_load8(m + i, (unsigned)min((size_t)8U, count - i), vec && i + 8U <= count, f);
        t += ns_squares(f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffU, t, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) t += sh[w];
        partial[(size_t)blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = t;
    }
}
template <typename T>
__global__ void __launch_bounds__(256)
ns_split_kernel(const T *__restrict__ g, const double *__restrict__ partial, int parts, __half *__restrict__ hi, __half *__restrict__ lo, unsigned rows, unsigned cols,
                unsigned octets, float eps, bool vec)
{
    gdb_pdl_sync();
    const T *m = g + (size_t)blockIdx.y * rows * cols;
    uint4 *h = reinterpret_cast<uint4 *>(hi) + (size_t)blockIdx.y * rows * octets, *l = reinterpret_cast<uint4 *>(lo) + (size_t)blockIdx.y * rows * octets;
    const size_t n = (size_t)rows * octets, stride = (size_t)gridDim.x * blockDim.x;
    size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    const auto load = [&](size_t k, float (&v)[8]) {
        const unsigned r = n < 0xffffffffU ? (unsigned)k / octets : (unsigned)(k / octets), c = (unsigned)(k - (size_t)r * octets) * 8U;
        if (c < cols) {
            ns_load8(m + (size_t)r * cols + c, cols - c, vec, v);
        } else {
            // (rows of the scratch are a multiple of 16 elements: the last octet may lie behind the matrix's row as a whole)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        }
    };
    // (the first elements are on their way while the partial sums are added, by every warp in the same order)
    float v[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (i + u * stride < n) load(i + u * stride, v[u]);
    }
    const int lane = threadIdx.x & 31;
    double part[NS_NORM_BLOCKS / 32], s = 0.0;
#pragma unroll
    for (int k = 0; k < NS_NORM_BLOCKS / 32; ++k) part[k] = lane + 32 * k < parts ? __ldg(&partial[(size_t)blockIdx.y * NS_NORM_BLOCKS + lane + 32 * k]) : 0.0;
#pragma unroll
    for (int k = 0; k < NS_NORM_BLOCKS / 32; ++k) s += part[k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffU, s, o);
    const double f = (double)NS_UP / (sqrt(s) + (double)eps);
    for (; i < n; i += 2U * stride) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const size_t k = i + u * stride;
            if (k >= n) break;
            uint4 a, b;
            ns_halves(v[u], f, (float)f, a, b);
            h[k] = a;
            l[k] = b;
            if (k + 2U * stride < n) load(k + 2U * stride, v[u]);
        }
    }
}

// ------------------------------------------------------------------ products
// GRAM: A = 2^-20 X X^T. POLY: P = b A + c A A. UPDATE: X <- a (hi + lo) + P hi. LAST: the same into the caller's tensor.
// A and P are symmetric (and commute with A), so the tiles on and above the diagonal are formed and those above it stored twice, and
// either order of the product's operands does.
enum { NS_GRAM, NS_POLY, NS_UPDATE, NS_LAST };

// Smaller sides up to which an FP16 result gets its full precision without being asked for it: operands as sums of two FP16 numbers, hi hi +
// hi lo + lo hi of three products in one accumulator. Rounded to one FP16 number each, A and P cost the result up to 1.7e-3 in the 2-norm
// where its singular values are close together (rounding errors of the diagonals add up), 3e-4 where a few stand out; with three products
// what is left is the result's own rounding, 2.1e-4. What they cost grows with the size and has no turn; the cut is where it is three
// quarters of a call. One product and three, one square matrix: 129 54 and 84 us (1.54 times), 256 63 and 106 (1.68), 448 81 and 140 (1.73),
// 480 83 and 147 (1.78), 512 87 and 152 (1.76), 640 94 and 173 (1.84), 896 117 and 233 (2.0); four of 5632 x 2048 1500 and 4010 (2.7). BF16
// results, whose own rounding is 1.7e-3 (2.1e-3 to 2.4e-3 with one product), keep one product unless asked (but where one launch does all,
// below, three take 6 to 13 us more of 25 to 60).
constexpr uint64_t NS_FINE = 448;

struct ns_maps {
    CUtensorMap a, b, a_lo, b_lo;   // operands
};
// What the epilogue reads and writes, [batch, M, pitch] with rows of a multiple of 32 bytes (LAST's output: dense, any alignment).
struct ns_shape {
    uint32_t M, N, K, tiles_m, tiles_n, batch, pitch;
    uint32_t parts;          // of a product: 1: hi hi; 3: hi hi + hi lo + lo hi, and A and P have low halves too
    float alpha, beta;
    const __half *in, *in_lo;   // POLY: A; UPDATE, LAST: X
    void *out;               // A, P, the next X, or the caller's tensor
    __half *out_lo;
    bool wide_out;           // LAST: the caller's rows take 32-byte stores
};

// One warp's piece of the result, 32 rows (a lane each) x COLS columns. Inputs and results go between registers and memory directly, 32 bytes a lane
// and access, beside the products' operands in shared memory, not through it: with tiles staged there for TMA a step's UPDATE of four 5632 x
// 2048 matrices took 170 us, without any epilogue traffic 128, and takes 153 so (tensor pipe 74 % busy, its reads of shared memory 34 % of
// what that delivers).
constexpr int NS_PIECE = 32, NS_STAGE_ROW = 80, NS_WARP_STAGE = NS_PIECE * NS_STAGE_ROW;   // rows of 64 bytes, 16 apart in the banks
template <int COLS> struct ns_row {
    uint32_t w[COLS / 2];
};
template <int COLS>
__device__ __forceinline__ void ns_load_row(ns_row<COLS> &r, const __half *p, uint32_t left)
{
#pragma unroll
    for (int k = 0; k < COLS / 16; ++k) {
        uint32_t *w = r.w + 8 * k;
        if (16U * k < left) {
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p + 16 * k)
                         : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 0U;
        }
    }
}
template <int COLS>
__device__ __forceinline__ void ns_store_row(void *base, const uint32_t *w, uint32_t left)
{
    __half *p = reinterpret_cast<__half *>(base);
#pragma unroll
    for (int k = 0; k < COLS / 16; ++k) {
        const uint32_t *v = w + 8 * k;
        if (16U * k < left) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + 16 * k), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                         "r"(v[6]), "r"(v[7])
                         : "memory");
        }
    }
}
// two numbers as sums of two FP16 ones each
__device__ __forceinline__ void ns_split2(float a, float b, uint32_t &hi, uint32_t &lo)
{
    hi = half_pack<__half>::pack(a, b);
    const float2 r = ns_two(hi);
    lo = half_pack<__half>::pack(a - r.x, b - r.y);
}
// the inputs of a piece, on their way while its products are formed
template <int MODE, int COLS>
__device__ __forceinline__ void ns_load_piece(ns_row<COLS> &in, ns_row<COLS> &lo, const ns_shape &sh, uint32_t row, uint32_t col0, uint32_t z)
{
    if (MODE == NS_GRAM) return;
    const uint32_t left = row < sh.M && col0 < sh.N ? sh.N - col0 : 0U;
    const size_t at = ((size_t)z * sh.M + (left != 0U ? row : 0U)) * sh.pitch + (left != 0U ? col0 : 0U);
    ns_load_row(in, sh.in + at, left);
    if (MODE != NS_POLY || sh.parts > 1U) ns_load_row(lo, sh.in_lo + at, left);
}
// the transposed piece: row e of it are the lanes' elements e
__device__ __forceinline__ void ns_store_mirrored(__half *out, const uint32_t *v, const ns_shape &sh, uint32_t row0, uint32_t col0, uint32_t z, unsigned char *stage, int lane)
{
#pragma unroll
    for (int e = 0; e < NS_PIECE; ++e) *reinterpret_cast<unsigned short *>(stage + e * NS_STAGE_ROW + lane * 2) = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
    __syncwarp();
    uint32_t w[NS_PIECE / 2];
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4 *>(w + 4 * j) = *reinterpret_cast<const uint4 *>(stage + lane * NS_STAGE_ROW + j * 16);
    const uint32_t row = col0 + lane, left = row < sh.M && row0 < sh.N ? sh.N - row0 : 0U;
    ns_store_row<NS_PIECE>(out + ((size_t)z * sh.M + row) * sh.pitch + row0, w, left);
    __syncwarp();
}
// v: the piece's accumulators. `stage` (this warp's): where a piece is transposed, or rows that take no 32-byte stores are put together.
template <int MODE, typename TOUT, int COLS>
__device__ __forceinline__ void ns_finish_piece(const ns_shape &sh, const ns_row<COLS> &in, ns_row<COLS> &lo, uint32_t (&v)[COLS], uint32_t row0, uint32_t col0, uint32_t z, bool mirror,
                                                unsigned char *stage, int lane)
{
    const uint32_t row = row0 + lane;
    const bool live = row < sh.M && col0 < sh.N;
    const uint32_t left = live ? sh.N - col0 : 0U;
    const size_t at = ((size_t)z * sh.M + row) * sh.pitch + col0;
#pragma unroll
    for (int e = 0; e < COLS / 2; ++e) {
        float f0 = sh.alpha * __uint_as_float(v[2 * e]), f1 = sh.alpha * __uint_as_float(v[2 * e + 1]);
        if (MODE != NS_GRAM) {
            float2 a = ns_two(in.w[e]);
            if (MODE != NS_POLY || sh.parts > 1U) {
                const float2 l = ns_two(lo.w[e]);
                a.x += l.x;
                a.y += l.y;
            }
            f0 = fmaf(sh.beta, a.x, f0);
            f1 = fmaf(sh.beta, a.y, f1);
        }
        if (MODE == NS_LAST) {
            v[e] = half_pack<TOUT>::pack(f0 * NS_DOWN, f1 * NS_DOWN);
        } else {
            if (MODE == NS_UPDATE || sh.parts > 1U) ns_split2(f0, f1, v[e], lo.w[e]); else v[e] = half_pack<__half>::pack(f0, f1);
        }
    }
    if (MODE == NS_LAST) {
        unsigned short *out = reinterpret_cast<unsigned short *>(sh.out) + ((size_t)z * sh.M + row0) * sh.N + col0;
        if (sh.wide_out) {
            ns_store_row<COLS>(out + (size_t)lane * sh.N, v, left);
        } else {
            const uint32_t rows = row0 < sh.M ? min(32U, sh.M - row0) : 0U;
#pragma unroll
            for (int h = 0; h < COLS / NS_PIECE; ++h) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t *w = v + h * (NS_PIECE / 2) + 4 * j;
                    *reinterpret_cast<uint4 *>(stage + lane * NS_STAGE_ROW + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                __syncwarp();
                const uint32_t c = h * NS_PIECE + lane;
                if (col0 + c < sh.N) {
#pragma unroll 8
                    for (uint32_t r = 0; r < rows; ++r) out[(size_t)r * sh.N + c] = *reinterpret_cast<const unsigned short *>(stage + r * NS_STAGE_ROW + lane * 2);
                }
                __syncwarp();
            }
        }
        return;
    }
    __half *out = reinterpret_cast<__half *>(sh.out);
    ns_store_row<COLS>(out + at, v, left);
    if (MODE == NS_UPDATE || sh.parts > 1U) ns_store_row<COLS>(sh.out_lo + at, lo.w, left);
    if constexpr (MODE != NS_UPDATE && COLS == NS_PIECE) {
        if (mirror) {
            ns_store_mirrored(out, v, sh, row0, col0, z, stage, lane);
            if (sh.parts > 1U) ns_store_mirrored(sh.out_lo, lo.w, sh, row0, col0, z, stage, lane);
        }
    }
}

// which of a product's parts a k step belongs to
__device__ __forceinline__ uint32_t ns_part(uint32_t it, uint32_t part_iters) { return (it >= part_iters ? 1U : 0U) + (it >= 2U * part_iters ? 1U : 0U); }

// ---- one CTA, one tile of 128 x BN: small matrices, where the number of SMs at work counts ----
// SPLIT: two CTAs of a cluster take half of the contraction each and send each other the sums of half of the tile's columns (GRAM of long
// matrices: few tiles, each a long chain of products).
constexpr int NS1_SENT_ROW = 144, NS1_SENT = BM * NS1_SENT_ROW;   // 32 FP32 sums of a row, rows 16 bytes apart in the banks
template <int BN, int STAGES, bool SPLIT> struct ns1_plan {
    static constexpr int STAGE_BYTES = (BM + BN) * BK * 2, WARPS = 4 * BN / NS_PIECE, THREADS = 64 + 32 * WARPS;
    static constexpr int SMEM = STAGES * STAGE_BYTES + WARPS * NS_WARP_STAGE + (SPLIT ? NS1_SENT : 0) + 256 + 1024;
    static_assert(BN == 32 || BN == 64, "columns of the operand's box");
};

template <bool A_MN, bool B_MN, int MODE, typename TOUT, int BN, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(ns1_plan<BN, STAGES, SPLIT>::THREADS)
ns_single_kernel(const __grid_constant__ ns_maps maps, const ns_shape sh, int *err_flag)
{
    typedef ns1_plan<BN, STAGES, SPLIT> plan;
    static_assert(!SPLIT || (MODE == NS_GRAM && BN == 64), "halves of 32 columns");
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    // UPDATE and LAST read X and its low half, which the launches before the preceding one wrote: their loads need not wait for it. The
    // operand that does is P.
    constexpr bool EARLY = !SYM, A_IS_X = !B_MN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023U) & ~(uintptr_t)1023U);
    unsigned char *staging = smem + STAGES * plan::STAGE_BYTES;
    unsigned char *sent = staging + plan::WARPS * NS_WARP_STAGE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sent + (SPLIT ? NS1_SENT : 0));   // full, empty, accumulator
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t z = blockIdx.y;
    uint32_t tm, tn;
    if (SYM) {
        // of row tile tm the column tiles from the diagonal on
        constexpr uint32_t STEP = BM / BN;
        uint32_t u = SPLIT ? blockIdx.x >> 1 : blockIdx.x;
        for (tm = 0; u >= sh.tiles_n - STEP * tm; ++tm) u -= sh.tiles_n - STEP * tm;
        tn = STEP * tm + u;
    } else {
        tm = blockIdx.x / sh.tiles_n;
        tn = blockIdx.x - tm * sh.tiles_n;
    }
    const uint32_t rank = SPLIT ? cluster_ctarank() : 0U, part_iters = (sh.K + BK - 1) / BK, all_iters = part_iters * sh.parts;
    const uint32_t first = rank * ((all_iters + 1U) / 2U), n_iters = SPLIT ? (rank == 0U ? (all_iters + 1U) / 2U : all_iters - first) : all_iters;
    const uint32_t m0 = tm * BM, n0 = tn * BN;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]), accum_bar = smem_u32(&bars[2 * STAGES]);
    auto load_a = [&](uint32_t it) {
        const uint32_t s = it % STAGES, dst = smem_u32(smem + s * plan::STAGE_BYTES), bar = full0 + 8 * s, p = ns_part(first + it, part_iters);
        const CUtensorMap *map = p == 2U ? &maps.a_lo : &maps.a;
        const int k0 = (int)((first + it - p * part_iters) * BK);
        if (A_MN) {
            tma_load_3d(dst, map, (int)m0, k0, (int)z, bar);
            tma_load_3d(dst + BK * 128, map, (int)m0 + 64, k0, (int)z, bar);
        } else {
            tma_load_3d(dst, map, k0, (int)m0, (int)z, bar);
        }
    };
    auto load_b = [&](uint32_t it) {
        const uint32_t s = it % STAGES, dst = smem_u32(smem + s * plan::STAGE_BYTES) + BM * BK * 2, bar = full0 + 8 * s, p = ns_part(first + it, part_iters);
        const CUtensorMap *map = p == 1U ? &maps.b_lo : &maps.b;
        const int k0 = (int)((first + it - p * part_iters) * BK);
        if (B_MN) tma_load_3d(dst, map, (int)n0, k0, (int)z, bar); else tma_load_3d(dst, map, k0, (int)n0, (int)z, bar);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2 * STAGES + 1; ++s) mbar_init(full0 + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncwarp();
    if (SPLIT) cluster_sync_all(); else __syncthreads();   // (the peer runs before its memory is written; under the end of the launch before)
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int quad = warp & 3, part = (warp - 2) >> 2;   // (epilogue warps: tensor-memory quadrant, columns)
    const uint32_t row0 = m0 + quad * 32, col0 = n0 + part * NS_PIECE;
    ns_row<NS_PIECE> in, lo;
    uint32_t v[NS_PIECE];
    bool ok = true;
    if (EARLY) {
        if (threadIdx.x == 0) {
            for (uint32_t it = 0; it < n_iters && it < STAGES; ++it) {
                mbar_expect_tx(full0 + 8 * it, plan::STAGE_BYTES);
                if (A_IS_X) load_a(it); else load_b(it);
            }
        } else if (warp >= 2) {
            ns_load_piece<MODE>(in, lo, sh, row0 + lane, col0, z);
        }
    }
    gdb_pdl_sync();

    if (warp == 0) {
        if (lane == 0) {
            for (uint32_t it = 0; it < n_iters; ++it) {
                const uint32_t s = it % STAGES, ph = (it / STAGES) & 1U;
                const bool begun = EARLY && it < STAGES;
                if (!begun) {
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1U)) {
                        atomicExch(err_flag, 701);
                        break;
                    }
                    mbar_expect_tx(full0 + 8 * s, plan::STAGE_BYTES);
                }
                if (!begun || !A_IS_X) load_a(it);
                if (!begun || A_IS_X) load_b(it);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t IDESC = (1U << 4) | ((A_MN ? 1U : 0U) << 15) | ((B_MN ? 1U : 0U) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            for (uint32_t it = 0; it < n_iters; ++it) {
                const uint32_t s = it % STAGES, ph = (it / STAGES) & 1U;
                if (!mbar_wait(full0 + 8 * s, ph)) {
                    atomicExch(err_flag, 702);
                    break;
                }
                tcgen05_fence_after();
                const uint32_t a_base = smem_u32(smem + s * plan::STAGE_BYTES), b_base = a_base + BM * BK * 2;
#pragma unroll
                for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                    const uint64_t adesc = A_MN ? make_smem_desc(a_base + kk * 2048, BK * 128, 1024) : make_smem_desc(a_base + kk * 32, 16, 1024);
                    const uint64_t bdesc = B_MN ? make_smem_desc(b_base + kk * 2048, BK * 128, 1024) : make_smem_desc(b_base + kk * 32, 16, 1024);
                    tcgen05_mma_f16(tmem_base, adesc, bdesc, IDESC, (it != 0 || kk != 0) ? 1U : 0U);
                }
                tcgen05_commit(empty0 + 8 * s);
            }
            tcgen05_commit(accum_bar);
        }
    } else {
        if (!EARLY) ns_load_piece<MODE>(in, lo, sh, row0 + lane, col0, z);
        ok = __all_sync(0xffffffffU, mbar_wait(accum_bar, 0));
        if (!ok && lane == 0) atomicExch(err_flag, 703);
        tcgen05_fence_after();
        if (ok) {
            tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(quad * 32) << 16) + part * NS_PIECE, v);
            if (SPLIT && part != (int)rank) {
                const uint32_t to = mapa_shared(smem_u32(sent) + (quad * 32 + lane) * NS1_SENT_ROW, rank ^ 1U);
#pragma unroll
                for (int k = 0; k < NS_PIECE; k += 4) {
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + 4 * k), "r"(v[k]), "r"(v[k + 1]), "r"(v[k + 2]), "r"(v[k + 3]) : "memory");
                }
            }
        }
    }
    if (SPLIT) {
        __syncwarp();
        cluster_sync_all();
        if (warp >= 2 && part == (int)rank) {
#pragma unroll
            for (int k = 0; k < NS_PIECE; k += 4) {
                const float4 o = *reinterpret_cast<const float4 *>(sent + (quad * 32 + lane) * NS1_SENT_ROW + 4 * k);
                v[k] = __float_as_uint(__uint_as_float(v[k]) + o.x);
                v[k + 1] = __float_as_uint(__uint_as_float(v[k + 1]) + o.y);
                v[k + 2] = __float_as_uint(__uint_as_float(v[k + 2]) + o.z);
                v[k + 3] = __float_as_uint(__uint_as_float(v[k + 3]) + o.w);
            }
        }
    }
    if (warp >= 2 && ok && (!SPLIT || part == (int)rank)) {
        ns_finish_piece<MODE, TOUT>(sh, in, lo, v, row0, col0, z, tn / (BM / BN) != tm, staging + (warp - 2) * NS_WARP_STAGE, lane);
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)BN) : "memory");
    }
}

// ---- a pair of CTAs, 256 x 256 tiles, persistent: tiles to fill the GPU. The roles and the two accumulators are those of
// gemm_tcgen05_pair.cu: each CTA fetches its own halves of the operands, the leader issues the products for both, the epilogue
// of one tile runs under the products of the next. ----
constexpr int NS2_BN = 256, NS2_STAGES = 5, NS2_WARPS = 8;
constexpr int NS2_STAGE_BYTES = (BM + NS2_BN / 2) * BK * 2;
constexpr int NS2_SMEM = NS2_STAGES * NS2_STAGE_BYTES + NS2_WARPS * NS_WARP_STAGE + 256 + 1024;

template <bool A_MN, bool B_MN, int MODE, typename TOUT>
__global__ void __launch_bounds__(32 * (2 + NS2_WARPS), 1)
ns_pair_kernel(const __grid_constant__ ns_maps maps, const ns_shape sh, int *err_flag)
{
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023U) & ~(uintptr_t)1023U);
    unsigned char *staging = smem + NS2_STAGES * NS2_STAGE_BYTES;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + NS2_WARPS * NS_WARP_STAGE);
    // full, empty, accumulator full [2], accumulator empty [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * NS2_STAGES + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
    const uint32_t part_iters = (sh.K + BK - 1) / BK, n_iters = part_iters * sh.parts;
    const uint32_t per = SYM ? sh.tiles_n * (sh.tiles_n + 1U) / 2U : sh.tiles_m * sh.tiles_n, units = per * sh.batch;
    auto tile_of = [&](uint32_t u, uint32_t &z, uint32_t &tm, uint32_t &tn) {
        z = u / per;
        u -= z * per;
        if (SYM) {
            for (tm = 0; u >= sh.tiles_n - tm; ++tm) u -= sh.tiles_n - tm;
            tn = tm + u;
        } else {
            tm = u / sh.tiles_n;
            tn = u - tm * sh.tiles_n;
        }
    };
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[NS2_STAGES]);
    const uint32_t tfull0 = smem_u32(&bars[2 * NS2_STAGES]), tempty0 = smem_u32(&bars[2 * NS2_STAGES + 2]);
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2 * NS2_STAGES + 2; ++s) mbar_init(full0 + 8 * s, 1);
        for (int b = 0; b < 2; ++b) mbar_init(tempty0 + 8 * b, 2 * NS2_WARPS);   // the epilogue warps of both CTAs
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)(2 * NS2_BN)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    gdb_pdl_sync();

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full_leader = mapa_shared(full0, 0);
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t u = cluster_id; u < units && ok; u += n_clusters) {
                uint32_t z, tm, tn;
                tile_of(u, z, tm, tn);
                const int am = (int)(tm * 2 * BM + rank * BM), bn = (int)(tn * NS2_BN + rank * (NS2_BN / 2));
                for (uint32_t kb = 0; kb < n_iters; ++kb, ++it) {
                    const uint32_t s = it % NS2_STAGES, ph = (it / NS2_STAGES) & 1U;
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1U)) {
                        atomicExch(err_flag, 711);
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * NS2_STAGE_BYTES);
                    const uint32_t a_dst = smem_u32(smem + s * NS2_STAGE_BYTES), b_dst = a_dst + BM * BK * 2, bar = full_leader + 8 * s;
                    const uint32_t p = ns_part(kb, part_iters);
                    const CUtensorMap *a = p == 2U ? &maps.a_lo : &maps.a, *b = p == 1U ? &maps.b_lo : &maps.b;
                    const int k0 = (int)((kb - p * part_iters) * BK);
                    if (A_MN) {
                        tma_load_3d_pair(a_dst, a, am, k0, (int)z, bar);
                        tma_load_3d_pair(a_dst + BK * 128, a, am + 64, k0, (int)z, bar);
                    } else {
                        tma_load_3d_pair(a_dst, a, k0, am, (int)z, bar);
                    }
                    if (B_MN) {
                        tma_load_3d_pair(b_dst, b, bn, k0, (int)z, bar);
                        tma_load_3d_pair(b_dst + BK * 128, b, bn + 64, k0, (int)z, bar);
                    } else {
                        tma_load_3d_pair(b_dst, b, k0, bn, (int)z, bar);
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t IDESC = (1U << 4) | ((A_MN ? 1U : 0U) << 15) | ((B_MN ? 1U : 0U) << 16) | ((uint32_t)(NS2_BN >> 3) << 17) | ((uint32_t)((2 * BM) >> 4) << 24);
            uint32_t it = 0, idx = 0;
            bool ok = true;
            for (uint32_t u = cluster_id; u < units && ok; u += n_clusters, ++idx) {
                const uint32_t buf = idx & 1U;
                if (!mbar_wait(tempty0 + 8 * buf, ((idx >> 1) & 1U) ^ 1U)) {
                    atomicExch(err_flag, 712);
                    break;
                }
                tcgen05_fence_after();
                const uint32_t d_tmem = tmem_base + buf * NS2_BN;
                for (uint32_t kb = 0; kb < n_iters; ++kb, ++it) {
                    const uint32_t s = it % NS2_STAGES, ph = (it / NS2_STAGES) & 1U;
                    if (!mbar_wait(full0 + 8 * s, ph)) {
                        atomicExch(err_flag, 713);
                        ok = false;
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t a_base = smem_u32(smem + s * NS2_STAGE_BYTES), b_base = a_base + BM * BK * 2;
#pragma unroll
                    for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                        const uint64_t adesc = A_MN ? make_smem_desc(a_base + kk * 2048, BK * 128, 1024) : make_smem_desc(a_base + kk * 32, 16, 1024);
                        const uint64_t bdesc = B_MN ? make_smem_desc(b_base + kk * 2048, BK * 128, 1024) : make_smem_desc(b_base + kk * 32, 16, 1024);
                        tcgen05_mma_f16_pair(d_tmem, adesc, bdesc, IDESC, (kb != 0 || kk != 0) ? 1U : 0U);
                    }
                    tcgen05_commit_pair(empty0 + 8 * s, 3);
                }
                if (ok) tcgen05_commit_pair(tfull0 + 8 * buf, 3);
            }
        }
    } else {
        // warps w and w + 4 share a tensor-memory quadrant and take half of the tile's columns each: in two pieces where whole lines of 128
        // bytes go to memory, in four square ones where they are transposed
        constexpr int COLS = SYM ? NS_PIECE : 64;
        const int quad = warp & 3, half = (warp - 2) >> 2;
        const uint32_t tempty_leader = mapa_shared(tempty0, 0);
        uint32_t idx = 0;
        for (uint32_t u = cluster_id; u < units; u += n_clusters, ++idx) {
            uint32_t z, tm, tn;
            tile_of(u, z, tm, tn);
            const uint32_t buf = idx & 1U, row0 = tm * 2 * BM + rank * BM + quad * 32, tbase = tmem_base + ((uint32_t)(quad * 32) << 16) + buf * NS2_BN + half * 128;
            const uint32_t first = tn * NS2_BN + half * 128;
            ns_row<COLS> in, lo;
            ns_load_piece<MODE>(in, lo, sh, row0 + lane, first, z);
            if (!__all_sync(0xffffffffU, mbar_wait(tfull0 + 8 * buf, (idx >> 1) & 1U))) {
                if (lane == 0) atomicExch(err_flag, 714);
                break;
            }
            tcgen05_fence_after();
#pragma unroll
            for (int p = 0; p < 128 / COLS; ++p) {
                if (p > 0) ns_load_piece<MODE>(in, lo, sh, row0 + lane, first + p * COLS, z);   // (two sets of registers, loaded a piece ahead, gained nothing)
                uint32_t v[COLS];
#pragma unroll
                for (int k = 0; k < COLS; k += 32) tmem_ld_32x32b_x32_nowait(tbase + p * COLS + k, *reinterpret_cast<uint32_t(*)[32]>(v + k));
                tmem_ld_wait();
                if ((p + 1) * COLS == 128) {
                    // the accumulator has been copied out
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(tempty_leader + 8 * buf);
                }
                ns_finish_piece<MODE, TOUT>(sh, in, lo, v, row0, first + p * COLS, z, tn != tm, staging + (warp - 2) * NS_WARP_STAGE, lane);
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tcgen05_fence_before();
    cluster_sync_all();   // neither CTA releases tensor memory while its peer may still use it
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)(2 * NS2_BN)) : "memory");
    }
}

// [batch, rows, cols] of 16-bit elements, boxes of box_rows x box_cols; `swizzle`: 128 bytes, else dense rows
bool ns_map(CUtensorMap *m, uint32_t dtype, const void *base, uint64_t batch, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows, uint32_t box_cols, bool swizzle)
{
    encode_tiled_fn fn = get_encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {cols, rows, batch}, strides[2] = {pitch * 2U, rows * pitch * 2U};
    const cuuint32_t box[3] = {box_cols, box_rows, 1}, estr[3] = {1, 1, 1};
    return fn(m, dtype == GDB_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct ns_tensor {       // a matrix of the scratch, as an operand and in the epilogue
    __half *p, *lo;
    uint64_t rows, cols, pitch;
};
bool ns_operand(CUtensorMap *m, const ns_tensor &t, const __half *p, uint64_t batch, bool mn, uint32_t tile)
{
    return mn ? ns_map(m, GDB_DTYPE_F16, p, batch, t.rows, t.cols, t.pitch, BK, 64, true) : ns_map(m, GDB_DTYPE_F16, p, batch, t.rows, t.cols, t.pitch, tile, BK, true);
}
// the maps of a product that comes again every step (or every second one), kept for the call
struct ns_memo {
    ns_maps maps;
    bool ready;
};

// ---- matrices whose smaller side is at most 128: all steps in one launch, a cluster of up to 16 CTAs per matrix ----
// A and P are one tile. Each CTA keeps up to 192 columns of X (rows for a tall matrix: X is taken transposed then) in shared memory, both
// halves, and forms its part of A; the parts are added over distributed shared memory (every CTA a share of the rows, then the sum to
// all), P is formed by every CTA for itself, and the CTA's columns are updated in place. Two exchanges a step in place of three launches
// that would each occupy a handful of SMs: 17 launches take the host 57 us alone.
constexpr int NT_M = 128, NT_W = 192, NT_W_ALONE = 256, NT_THREADS = 512, NT_WARPS = NT_THREADS / 32, NT_MAX_CTAS = 16;
constexpr int NT_X_BYTES = NT_M * NT_W * 2, NT_X_BYTES_ALONE = NT_M * NT_W_ALONE * 2, NT_A_BYTES = NT_M * NT_M * 2, NT_PARTS = NT_M * NT_M * 4;
constexpr int NT_SMEM = 2 * NT_X_BYTES + 2 * NT_A_BYTES + NT_PARTS + 512 + 1024;   // (one alone has no parts)
static_assert(2 * NT_X_BYTES_ALONE <= 2 * NT_X_BYTES + NT_PARTS, "room for the columns of one CTA");

// element (row, col) of a tile of 128 rows in blocks of 64 columns, 128-byte swizzle: the 16 bytes that hold columns 8 * octet ...
__device__ __forceinline__ uint32_t nt_at(uint32_t row, uint32_t octet) { return (octet >> 3) * (NT_M * 128U) + row * 128U + (((octet & 7U) ^ (row & 7U)) << 4); }
__device__ __forceinline__ void nt_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }

template <typename T, typename TOUT>
__global__ void __launch_bounds__(NT_THREADS, 1)
ns_tile_kernel(const T *__restrict__ g, TOUT *out, uint32_t rows, uint32_t cols, uint32_t steps, float ca, float cb, float cc, float eps, bool vec, bool vec_out, int *err_flag)
{
    gdb_pdl_sync();
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023U) & ~(uintptr_t)1023U);
    const uint32_t rank = cluster_ctarank(), ctas = gridDim.x, z = blockIdx.y;   // (one cluster per matrix: grid.x is its size)
    unsigned char *sa = smem, *sl = sa + NT_A_BYTES, *xh = sl + NT_A_BYTES, *xl = xh + (ctas == 1U ? NT_X_BYTES_ALONE : NT_X_BYTES),   // A (then P) and X, hi and lo each
                  *parts = smem + 2 * NT_A_BYTES + 2 * NT_X_BYTES;                                                                         // parts of A
    double *sums = reinterpret_cast<double *>(parts + NT_PARTS);                                        // [CTAs], then the warps' sums
    uint64_t *bar = reinterpret_cast<uint64_t *>(sums + NT_MAX_CTAS + NT_WARPS);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar + 3);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool tall = rows > cols;
    const uint32_t m = tall ? cols : rows, n = tall ? rows : cols;
    const uint32_t width = ((n + ctas - 1U) / ctas + 63U) & ~63U, j0 = rank * width;   // columns of X here (multiples of 64)
    const uint32_t done = smem_u32(bar), got_parts = done + 8U, got_sum = done + 16U;
    if (threadIdx.x == 0) {
        for (int k = 0; k < 3; ++k) mbar_init(done + 8 * k, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512U) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // eight columns of a row: contiguous in memory, or one from each of eight rows of a tall matrix (neighbouring threads take
    // neighbouring elements of those). A thread visits the same octets when it loads, splits and stores.
    const uint32_t octets = width / 8U;
    auto place = [&](uint32_t i, uint32_t &row, uint32_t &octet) {
        row = tall ? i % NT_M : i / octets;
        octet = tall ? i / NT_M : i % octets;
    };
    const T *x = g + (size_t)z * rows * cols;
    double t = 0.0;
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < NT_M * octets; i += NT_THREADS) {
        uint32_t row, octet;
        place(i, row, octet);
        const uint32_t j = j0 + octet * 8U;
        float f[8];
        if (row >= m || j >= n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = 0.0f;
        } else if (tall) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = j + e < n ? gdb_io<T>::ld(x, (size_t)(j + e) * cols + row) : 0.0f;
        } else {
            ns_load8(x + (size_t)row * cols + j, n - j, vec, f);
        }
        t += ns_squares(f);
        // as they are, four and four in the places of the two halves
        *reinterpret_cast<float4 *>(xh + nt_at(row, octet)) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4 *>(xl + nt_at(row, octet)) = make_float4(f[4], f[5], f[6], f[7]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffU, t, o);
    if (lane == 0) sums[NT_MAX_CTAS + warp] = t;
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;   // columns 0..255: X, 256..383: A, 384..511: A A
    cluster_sync_all();                 // (every CTA of the cluster runs before its memory is written)
    if (threadIdx.x < ctas) {
        double s = 0.0;
        for (int w = 0; w < NT_WARPS; ++w) s += sums[NT_MAX_CTAS + w];
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(mapa_shared(smem_u32(sums + rank), threadIdx.x)), "l"(__double_as_longlong(s)) : "memory");
    }
    __syncwarp();
    cluster_sync_all();
    double norm = 0.0;
    for (uint32_t r = 0; r < ctas; ++r) norm += sums[r];
    const double factor = (double)NS_UP / (sqrt(norm) + (double)eps);
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < NT_M * octets; i += NT_THREADS) {
        uint32_t row, octet;
        place(i, row, octet);
        const float4 a = *reinterpret_cast<const float4 *>(xh + nt_at(row, octet)), b = *reinterpret_cast<const float4 *>(xl + nt_at(row, octet));
        const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        ns_halves(f, factor, (float)factor, *reinterpret_cast<uint4 *>(xh + nt_at(row, octet)), *reinterpret_cast<uint4 *>(xl + nt_at(row, octet)));
    }

    // a thread's row of A, P and X (tensor-memory lane) and its columns: 32 of every 128
    const int quad = warp & 3, part = warp >> 2;
    const uint32_t row = quad * 32 + lane, tlane = (uint32_t)(quad * 32) << 16;
    const uint32_t share = NT_M / ctas;   // rows of A that this CTA adds up
    constexpr float DOWN2 = NS_DOWN * NS_DOWN;
    uint32_t phase = 0;
    bool ok = true;
    // the products of a phase, hi hi + hi lo + lo hi, by one thread, and the wait for them by all
    auto products = [&](uint32_t d, const unsigned char *a_hi, const unsigned char *a_lo, const unsigned char *b_hi, const unsigned char *b_lo, bool b_mn, uint32_t n_cols,
                        uint32_t blocks, uint32_t block_bytes) {
        nt_fence();
        tcgen05_fence_before();
        __syncthreads();
        if (threadIdx.x == 0) {
            tcgen05_fence_after();
            const uint32_t idesc = (1U << 4) | ((b_mn ? 1U : 0U) << 16) | ((n_cols >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            for (uint32_t q = 0; q < 3U; ++q) {
                const uint32_t a = smem_u32(q == 2U ? a_lo : a_hi), b = smem_u32(q == 1U ? b_lo : b_hi);
                for (uint32_t k = 0; k < blocks; ++k) {
                    for (uint32_t kk = 0; kk < BK / UMMA_K; ++kk) {
                        const uint64_t ad = make_smem_desc(a + k * (NT_M * 128U) + kk * 32, 16, 1024);
                        const uint64_t bd = b_mn ? make_smem_desc(b + k * block_bytes + kk * 2048, NT_M * 128U, 1024) : make_smem_desc(b + k * block_bytes + kk * 32, 16, 1024);
                        tcgen05_mma_f16(d, ad, bd, idesc, (q != 0 || k != 0 || kk != 0) ? 1U : 0U);
                    }
                }
            }
            tcgen05_commit(done);
        }
        if (ok && !mbar_wait(done, phase)) {
            ok = false;
            atomicExch(err_flag, 721);
        }
        phase ^= 1U;
        __syncwarp();
        tcgen05_fence_after();
    };
    for (uint32_t step = 0; step < steps; ++step) {
        // this CTA's part of A = X X^T
        products(tmem + 256U, xh, xl, xh, xl, false, NT_M, width / BK, NT_M * 128U);
        uint32_t v[32];
        tmem_ld_32x32b_x32(tmem + tlane + 256U + part * 32, v);
        if (ctas > 1U) {
            // Sent with their completion counted at the receiver, 64 KB of parts and as many of sums a step. Nobody is overrun: parts
            // of the next step are sent by those who have all of this step's sums, sums by those who have all parts.
            if (threadIdx.x == 0) {
                mbar_expect_tx(got_parts, NT_PARTS);
                mbar_expect_tx(got_sum, 2 * NT_A_BYTES);
            }
            const uint32_t to = mapa_shared(smem_u32(parts) + (rank * share + row % share) * 512U, row / share), to_bar = mapa_shared(got_parts, row / share);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t at = to + (((uint32_t)(part * 8 + k) ^ (row & 7U)) << 4);
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at), "r"(v[4 * k]), "r"(v[4 * k + 1]),
                             "r"(v[4 * k + 2]), "r"(v[4 * k + 3]), "r"(to_bar)
                             : "memory");
            }
            if (ok && !mbar_wait(got_parts, step & 1U)) {
                ok = false;
                atomicExch(err_flag, 722);
            }
            for (uint32_t i = threadIdx.x; i < share * 32U; i += NT_THREADS) {
                const uint32_t r = i / 32U, c4 = i % 32U, to_row = rank * share + r;
                float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (uint32_t k = 0; k < ctas; ++k) {
                    const float4 p = *reinterpret_cast<const float4 *>(parts + (k * share + r) * 512U + ((c4 ^ (r & 7U)) << 4));
                    s.x += p.x;
                    s.y += p.y;
                    s.z += p.z;
                    s.w += p.w;
                }
                uint32_t w[4];   // hi, hi, lo, lo
                ns_split2(s.x * DOWN2, s.y * DOWN2, w[0], w[2]);
                ns_split2(s.z * DOWN2, s.w * DOWN2, w[1], w[3]);
                const uint32_t at = smem_u32(sa) + nt_at(to_row, c4 >> 1) + (c4 & 1U) * 8U;
                for (uint32_t k = 0; k < ctas; ++k) {
                    const uint32_t dst = (rank + k) % ctas;
                    const uint32_t to_sum = mapa_shared(at, dst), to_bar = mapa_shared(got_sum, dst);
                    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to_sum), "r"(w[0]), "r"(w[1]), "r"(to_bar) : "memory");
                    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to_sum + (uint32_t)NT_A_BYTES), "r"(w[2]), "r"(w[3]),
                                 "r"(to_bar)
                                 : "memory");
                }
            }
            if (ok && !mbar_wait(got_sum, step & 1U)) {
                ok = false;
                atomicExch(err_flag, 723);
            }
            __syncwarp();
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t w[4], l[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) ns_split2(__uint_as_float(v[8 * k + 2 * e]) * DOWN2, __uint_as_float(v[8 * k + 2 * e + 1]) * DOWN2, w[e], l[e]);
                *reinterpret_cast<uint4 *>(sa + nt_at(row, part * 4 + k)) = make_uint4(w[0], w[1], w[2], w[3]);
                *reinterpret_cast<uint4 *>(sl + nt_at(row, part * 4 + k)) = make_uint4(l[0], l[1], l[2], l[3]);
            }
        }
        // P = b A + c A A in the place of A (which is symmetric: rows serve as columns). The other CTAs write the next A there only after
        // this one has sent its next part, behind the products that read P.
        products(tmem + 384U, sa, sl, sa, sl, false, NT_M, 2U, NT_M * 128U);
        tmem_ld_32x32b_x32(tmem + tlane + 384U + part * 32, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t at = nt_at(row, part * 4 + k);
            const uint4 a = *reinterpret_cast<const uint4 *>(sa + at), b = *reinterpret_cast<const uint4 *>(sl + at);
            uint32_t w[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = ns_two((&a.x)[e]), r = ns_two((&b.x)[e]);
                ns_split2(fmaf(cb, f.x + r.x, cc * __uint_as_float(v[8 * k + 2 * e])), fmaf(cb, f.y + r.y, cc * __uint_as_float(v[8 * k + 2 * e + 1])), w[e], l[e]);
            }
            *reinterpret_cast<uint4 *>(sa + at) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4 *>(sl + at) = make_uint4(l[0], l[1], l[2], l[3]);
        }
        // X <- a X + P X, this CTA's columns
        products(tmem, sa, sl, xh, xl, true, width, 2U, BK * 128U);
        const bool last = step + 1U == steps;
        const f32x2 ca2 = f2_make(ca, ca);
#pragma unroll 1
        for (uint32_t c = part * 32U; c < width; c += 128U) {
            tmem_ld_32x32b_x32(tmem + tlane + c, v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t at = nt_at(row, c / 8U + k);
                const uint4 h = *reinterpret_cast<const uint4 *>(xh + at), l = *reinterpret_cast<const uint4 *>(xl + at);
                uint4 nh, nl = make_uint4(0U, 0U, 0U, 0U);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 a = ns_two((&h.x)[e]), b = ns_two((&l.x)[e]);
                    float f0, f1;
                    f2_split(f2_fma(ca2, f2_add(f2_make(a.x, a.y), f2_make(b.x, b.y)), f2_make(__uint_as_float(v[8 * k + 2 * e]), __uint_as_float(v[8 * k + 2 * e + 1]))), f0, f1);
                    if (last) {
                        (&nh.x)[e] = half_pack<TOUT>::pack(f0 * NS_DOWN, f1 * NS_DOWN);
                    } else {
                        ns_split2(f0, f1, (&nh.x)[e], (&nl.x)[e]);
                    }
                }
                *reinterpret_cast<uint4 *>(xh + at) = nh;
                if (!last) *reinterpret_cast<uint4 *>(xl + at) = nl;
            }
        }
    }
    // the result lies in the place of hi
    __syncthreads();
    TOUT *o = out + (size_t)z * rows * cols;
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < NT_M * octets; i += NT_THREADS) {
        uint32_t r, octet;
        place(i, r, octet);
        const uint32_t j = j0 + octet * 8U;
        if (r >= m || j >= n) continue;
        const uint4 w = *reinterpret_cast<const uint4 *>(xh + nt_at(r, octet));
        if (!tall && vec_out) {
            *reinterpret_cast<uint4 *>(o + (size_t)r * cols + j) = w;
            continue;
        }
        unsigned short *p = reinterpret_cast<unsigned short *>(o) + (tall ? (size_t)j * cols + r : (size_t)r * cols + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (j + e < n) p[tall ? (size_t)e * cols : (size_t)e] = (unsigned short)((&w.x)[e >> 1] >> (16 * (e & 1)));
        }
    }
    __syncwarp();
    tcgen05_fence_before();
    cluster_sync_all();
    if (warp == 0) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512U) : "memory");
    }
}

template <typename T, typename TOUT>
gd_status ns_launch_tile(gd_backend *be, const void *g, void *out, const gdb200_orthogonalize_args *a)
{
    auto kern = ns_tile_kernel<T, TOUT>;
    static bool ready = false;
    if (!ready) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NT_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return gdb_fail(be, e, "orthogonalize attributes");
        ready = true;
    }
    const uint64_t n = std::max(a->rows, a->cols);
    unsigned ctas = 1;
    // Enough CTAs for the columns, and more, down to 64 columns each, while all matrices' CTAs run at once: the rows of A that each adds up
    // and sends get fewer (16 x 300: two CTAs 72 us, four 64, eight 60; 128 x 1400: eight 74, sixteen 72).
    if (n > NT_W_ALONE) {
        while (ctas * NT_W < n || (ctas < NT_MAX_CTAS && ctas * 64U < n && 2U * ctas * a->batch <= gdb_usable_sms(be))) ctas *= 2U;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // see gdb_pdl_sync()
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(ctas, (unsigned)a->batch);
    cfg.blockDim = dim3(NT_THREADS);
    cfg.dynamicSmemBytes = NT_SMEM;
    cfg.stream = be->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const bool vec = a->cols % 8U == 0U && (uintptr_t)g % 16U == 0U;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (const T *)g, (TOUT *)out, (uint32_t)a->rows, (uint32_t)a->cols, a->steps, a->a, a->b, a->c, a->eps, vec,
                                             a->cols % 8U == 0U && (uintptr_t)out % 16U == 0U, be->err_flag);
    if (e != cudaSuccess) {
        be->launches += 1U;
        return gdb_fail(be, e, "orthogonalize tile");
    }
    return gdb_launched(be, "orthogonalize tile");
}

// a launch of clusters of two
template <typename K>
gd_status ns_launch_clusters(gd_backend *be, K kern, dim3 grid, unsigned threads, int smem, const ns_maps &maps, const ns_shape &sh)
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // see gdb_pdl_sync()
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = be->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, maps, sh, be->err_flag);
    if (e != cudaSuccess) {
        be->launches += 1U;
        return gdb_fail(be, e, "orthogonalize product");
    }
    return gdb_launched(be, "orthogonalize product");
}

template <bool A_MN, bool B_MN, int MODE, typename TOUT, int BN, bool SPLIT = false>
gd_status ns_launch_single(gd_backend *be, const ns_maps &maps, const ns_shape &sh, uint32_t tiles)
{
    // UPDATE and LAST: two CTAs fit an SM, or one beside a CTA of the preceding POLY
    constexpr int STAGES = MODE == NS_GRAM || MODE == NS_POLY ? (BN == 32 ? 5 : 4) : (BN == 32 ? 4 : 3);
    typedef ns1_plan<BN, STAGES, SPLIT> plan;
    auto kern = ns_single_kernel<A_MN, B_MN, MODE, TOUT, BN, STAGES, SPLIT>;
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, plan::SMEM);
        if (e != cudaSuccess) return gdb_fail(be, e, "orthogonalize smem attribute");
        ready = true;
    }
    if (SPLIT) return ns_launch_clusters(be, kern, dim3(2U * tiles, sh.batch), plan::THREADS, plan::SMEM, maps, sh);
    gdb_launch(kern, dim3(tiles, sh.batch), plan::THREADS, plan::SMEM, be->stream, maps, sh, be->err_flag);
    return gdb_launched(be, "orthogonalize product");
}

template <bool A_MN, bool B_MN, int MODE, typename TOUT>
gd_status ns_launch_pair(gd_backend *be, const ns_maps &maps, const ns_shape &sh, uint32_t units)
{
    auto kern = ns_pair_kernel<A_MN, B_MN, MODE, TOUT>;
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS2_SMEM);
        if (e != cudaSuccess) return gdb_fail(be, e, "orthogonalize smem attribute");
        ready = true;
    }
    const uint32_t most = gdb_usable_sms(be) / 2U;
    return ns_launch_clusters(be, kern, dim3(2U * (units < most ? units : most)), 32U * (2 + NS2_WARPS), NS2_SMEM, maps, sh);
}

// One product of a step: operands xa and xb; sh has what the epilogue needs.
template <bool A_MN, bool B_MN, int MODE, typename TOUT = __half>
gd_status ns_product(gd_backend *be, const ns_tensor &xa, const ns_tensor &xb, ns_shape sh, ns_memo *memo)
{
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    const uint64_t sms = gdb_usable_sms(be), clusters = sms / 2U;
    const uint32_t p_m = (sh.M + 255U) / 256U, p_n = (sh.N + 255U) / 256U, s_m = (sh.M + 127U) / 128U;
    const uint32_t pairs = (SYM ? p_n * (p_n + 1U) / 2U : p_m * p_n) * sh.batch;
    auto singles = [&](uint32_t bn) {
        const uint32_t s_n = (sh.N + bn - 1U) / bn, step = 128U / bn;
        uint32_t n = s_m * s_n;
        if (SYM) {
            n = 0;
            for (uint32_t i = 0; step * i < s_n; ++i) n += s_n - step * i;
        }
        return n;
    };
    // Time of a launch in units of 10 ns, as measured: a fixed part (dependency on the launch before, first operands, epilogue), one per
    // k step of 64 and round of tiles (the operands' way into shared memory), and what a further round adds where one CTA per SM starts
    // anew. One call on a 512 x 512, 1024 x 1024, 2048 x 2048 matrix: pair 182, 221, 322 us, 128 x 64 tiles 91, 134, 411 us, 128 x 32
    // tiles 83, 123, 413 us.
    const uint32_t wide = singles(64), narrow = B_MN ? 0U : singles(32), iters = (sh.K + BK - 1U) / BK * sh.parts;
    auto cost = [&](uint64_t fixed, uint64_t again, uint64_t step, uint64_t tiles, uint64_t places, uint64_t its) {
        const uint64_t rounds = (tiles + places - 1U) / places;
        return fixed + again * (rounds - 1U) + step * its * rounds;
    };
    const uint64_t none = UINT64_MAX, again = SYM ? 250U : 80U, c_pair = cost(900, 100, 39, pairs, clusters, iters),
                   c_wide = cost(320, again, 35, (uint64_t)wide * sh.batch, sms, iters), c_narrow = B_MN ? none : cost(285, again, 33, (uint64_t)narrow * sh.batch, sms, iters),
                   c_split = MODE == NS_GRAM && iters > 1U ? cost(530, again, 35, 2U * (uint64_t)wide * sh.batch, sms, (iters + 1U) / 2U) : none;
    const uint64_t least = std::min(std::min(c_pair, c_wide), std::min(c_narrow, c_split));
    const bool pair = c_pair == least, split = !pair && c_split == least, slim = !pair && !split && c_narrow == least;
    const uint32_t bn = pair ? 256U : (slim ? 32U : 64U);
    sh.tiles_m = pair ? p_m : s_m;
    sh.tiles_n = (sh.N + bn - 1U) / bn;
    ns_maps &maps = memo->maps;   // (UPDATE's and LAST's tiles are the same)
    if (!memo->ready) {
        const uint32_t box = pair ? 128U : bn;
        if (!ns_operand(&maps.a, xa, xa.p, sh.batch, A_MN, 128) || !ns_operand(&maps.b, xb, xb.p, sh.batch, B_MN, box)) return GD_ERR_UNSUPPORTED;
        if (sh.parts > 1U && (!ns_operand(&maps.a_lo, xa, xa.lo, sh.batch, A_MN, 128) || !ns_operand(&maps.b_lo, xb, xb.lo, sh.batch, B_MN, box))) return GD_ERR_UNSUPPORTED;
        memo->ready = true;
    }
    if (pair) return ns_launch_pair<A_MN, B_MN, MODE, TOUT>(be, maps, sh, pairs);
    if constexpr (!B_MN) {
        if (slim) return ns_launch_single<A_MN, B_MN, MODE, TOUT, 32>(be, maps, sh, narrow);
    }
    if constexpr (MODE == NS_GRAM) {
        if (split) return ns_launch_single<A_MN, B_MN, MODE, TOUT, 64, true>(be, maps, sh, wide);
    }
    return ns_launch_single<A_MN, B_MN, MODE, TOUT, 64>(be, maps, sh, wide);
}

// Where the parts of the scratch lie: the iterate's high halves (two, used in turn), its low halves, A's and P's, the sums of squares.
struct ns_layout {
    size_t small, pitch, small_pitch;
    uint32_t parts;
    size_t hi[2], lo[2], gram, gram_lo, poly, poly_lo, norm, total;
};
bool ns_plan(const gdb200_orthogonalize_args *a, ns_layout *l)
{
    if (a == NULL || a->rows >= (1U << 24) || a->cols >= (1U << 24) || a->batch > 65535U || a->pairs > 1U) return false;
    l->small = a->rows < a->cols ? a->rows : a->cols;
    l->pitch = (a->cols + 15U) & ~(uint64_t)15U;   // (32 bytes: one access of the epilogue)
    l->small_pitch = (l->small + 15U) & ~(size_t)15U;
    // (the products count tiles of a batch in 32 bits)
    if ((a->rows / 128U + 1U) * (a->cols / 64U + 1U) * (a->batch + 1U) > 0x7fffffffU) return false;
    const size_t x = (a->batch * a->rows * l->pitch * 2U + 255U) & ~(size_t)255U, s = (a->batch * l->small * l->small_pitch * 2U + 255U) & ~(size_t)255U;
    l->parts = a->pairs != 0U || l->small <= NS_FINE ? 3U : 1U;
    const size_t s_lo = l->parts > 1U ? s : 0U;
    size_t at = 0U;
    const auto next = [&](size_t *where, size_t bytes) {
        *where = at;
        at += bytes;
    };
    next(&l->hi[0], x);
    next(&l->hi[1], x);
    next(&l->lo[0], x);
    if (l->parts > 1U) next(&l->lo[1], x); else l->lo[1] = l->lo[0];   // (an operand of other CTAs' products too, or read and written in place)
    next(&l->gram, s);
    next(&l->gram_lo, s_lo);
    next(&l->poly, s);
    next(&l->poly_lo, s_lo);
    next(&l->norm, a->batch * NS_NORM_BLOCKS * sizeof(double));
    l->total = at;
    return true;
}

template <typename T>
gd_status first_iterate(gd_backend *be, const void *g, double *partial, __half *hi, __half *lo, const gdb200_orthogonalize_args *a, size_t pitch)
{
    const size_t count = a->rows * a->cols;
    const bool even = (uintptr_t)g % 16U == 0U;
    const size_t want = (count + 4095U) / 4096U, most = (size_t)be->sm_count * 8U / a->batch + 1U;
    size_t parts = want < most ? want : most;
    if (parts > NS_NORM_BLOCKS) parts = NS_NORM_BLOCKS;
    gdb_launch(ns_norm_kernel<T>, dim3((unsigned)parts, (unsigned)a->batch), 256, 0, be->stream, (const T *)g, partial, count, even && (a->batch == 1U || count % 8U == 0U));
    gd_status st = gdb_launched(be, "orthogonalize norm");
    if (st != GD_OK) return st;
    // (one wave of blocks, at six an SM, over all matrices)
    const unsigned split_most = (unsigned)(((uint64_t)be->sm_count * 6U + a->batch - 1U) / a->batch), split_want = gdb_grid_for(a->rows * (pitch / 8U), 256, be, 6);
    gdb_launch(ns_split_kernel<T>, dim3(split_want < split_most ? split_want : split_most, (unsigned)a->batch), 256, 0, be->stream, (const T *)g, (const double *)partial, (int)parts, hi, lo,
               (unsigned)a->rows, (unsigned)a->cols, (unsigned)(pitch / 8U), a->eps, even && a->cols % 8U == 0U);
    return gdb_launched(be, "orthogonalize split");
}

}  // namespace

extern "C" {

size_t gdb200_orthogonalize_scratch_bytes(const gdb200_orthogonalize_args *args)
{
    ns_layout l;
    return ns_plan(args, &l) ? l.total : 0U;
}

gd_status gdb200_orthogonalize(gd_backend *be, const gd_backend_tensor_view *x, const gd_backend_tensor_view *out, const gd_backend_tensor_view *scratch,
                               const gdb200_orthogonalize_args *a)
{
    if (be == NULL || x == NULL || out == NULL || scratch == NULL || a == NULL || a->steps == 0U || !(a->eps >= 0.0f) || a->pairs > 1U) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    ns_layout l;
    if (!gdb_is_float_dtype(x->dtype) || (out->dtype != GDB_DTYPE_F16 && out->dtype != GDB_DTYPE_BF16) || scratch->dtype != GDB_DTYPE_U8 || !ns_plan(a, &l)) {
        return GD_ERR_UNSUPPORTED;
    }
    const size_t count = a->batch * a->rows * a->cols;
    const void *xp = gdb_tv_ptr(x, x->dtype);
    void *op = gdb_tv_ptr(out, out->dtype);
    unsigned char *sp = (unsigned char *)gdb_tv_ptr(scratch, GDB_DTYPE_U8);
    if (xp == NULL || op == NULL || sp == NULL || x->count != count || out->count != count || scratch->count < l.total || ((uintptr_t)sp % 256U) != 0U) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (count == 0U) {
        return GD_OK;
    }
    const uint64_t rows = a->rows, cols = a->cols, m = l.small;
    if (m <= NT_M && std::max(rows, cols) <= (uint64_t)NT_W * NT_MAX_CTAS) {
        const bool half_out = out->dtype == GDB_DTYPE_F16;
        if (x->dtype == GDB_DTYPE_F16) return half_out ? ns_launch_tile<__half, __half>(be, xp, op, a) : ns_launch_tile<__half, __nv_bfloat16>(be, xp, op, a);
        if (x->dtype == GDB_DTYPE_BF16) return half_out ? ns_launch_tile<__nv_bfloat16, __half>(be, xp, op, a) : ns_launch_tile<__nv_bfloat16, __nv_bfloat16>(be, xp, op, a);
        return half_out ? ns_launch_tile<float, __half>(be, xp, op, a) : ns_launch_tile<float, __nv_bfloat16>(be, xp, op, a);
    }
    const bool tall = rows > cols;
    const auto half_at = [&](size_t at) { return (__half *)(sp + at); };
    const ns_tensor xs[2] = {{half_at(l.hi[0]), half_at(l.lo[0]), rows, cols, l.pitch}, {half_at(l.hi[1]), half_at(l.lo[1]), rows, cols, l.pitch}};
    const ns_tensor gram = {half_at(l.gram), half_at(l.gram_lo), m, m, l.small_pitch}, poly = {half_at(l.poly), half_at(l.poly_lo), m, m, l.small_pitch};
    ns_memo grams[2], polys, updates[2];
    for (ns_memo *p : {&grams[0], &grams[1], &polys, &updates[0], &updates[1]}) p->ready = false;
    double *norm = (double *)(sp + l.norm);
    gd_status st = x->dtype == GDB_DTYPE_F16    ? first_iterate<__half>(be, xp, norm, xs[0].p, xs[0].lo, a, l.pitch)
                   : x->dtype == GDB_DTYPE_BF16 ? first_iterate<__nv_bfloat16>(be, xp, norm, xs[0].p, xs[0].lo, a, l.pitch)
                                                : first_iterate<float>(be, xp, norm, xs[0].p, xs[0].lo, a, l.pitch);
    for (uint32_t k = 0; k < a->steps && st == GD_OK; ++k) {
        const ns_tensor &x0 = xs[k & 1U], &x1 = xs[(k & 1U) ^ 1U];
        ns_shape square = {};
        square.parts = out->dtype == GDB_DTYPE_F16 || a->pairs != 0U || m <= (uint64_t)NT_M ? l.parts : 1U;   // (up to NT_M as in the one launch of shorter matrices)
        square.M = square.N = (uint32_t)m;
        square.K = (uint32_t)(tall ? rows : cols);
        square.batch = (uint32_t)a->batch;
        square.alpha = NS_DOWN * NS_DOWN;
        square.pitch = (uint32_t)l.small_pitch;
        square.out = gram.p;
        square.out_lo = gram.lo;
        st = tall ? ns_product<true, true, NS_GRAM>(be, x0, x0, square, &grams[k & 1U]) : ns_product<false, false, NS_GRAM>(be, x0, x0, square, &grams[k & 1U]);
        if (st != GD_OK) break;
        square.K = (uint32_t)m;
        square.alpha = a->c;
        square.beta = a->b;
        square.in = gram.p;
        square.in_lo = gram.lo;
        square.out = poly.p;
        square.out_lo = poly.lo;
        st = ns_product<false, false, NS_POLY>(be, gram, gram, square, &polys);
        if (st != GD_OK) break;
        ns_shape full = square;
        full.M = (uint32_t)rows;
        full.N = (uint32_t)cols;
        full.pitch = (uint32_t)l.pitch;
        full.alpha = 1.0f;
        full.beta = a->a;
        full.in = x0.p;
        full.in_lo = x0.lo;
        if (k + 1U < a->steps) {
            full.out = x1.p;
            full.out_lo = x1.lo;
            st = tall ? ns_product<false, false, NS_UPDATE>(be, x0, poly, full, &updates[k & 1U]) : ns_product<false, true, NS_UPDATE>(be, poly, x0, full, &updates[k & 1U]);
        } else {
            full.out = op;
            full.wide_out = cols % 16U == 0U && (uintptr_t)op % 32U == 0U;
            if (out->dtype == GDB_DTYPE_F16) st = tall ? ns_product<false, false, NS_LAST, __half>(be, x0, poly, full, &updates[k & 1U]) : ns_product<false, true, NS_LAST, __half>(be, poly, x0, full, &updates[k & 1U]);
            else st = tall ? ns_product<false, false, NS_LAST, __nv_bfloat16>(be, x0, poly, full, &updates[k & 1U]) : ns_product<false, true, NS_LAST, __nv_bfloat16>(be, poly, x0, full, &updates[k & 1U]);
        }
    }
    return st;
}

}  // extern "C"
