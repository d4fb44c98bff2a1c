// Orthogonalisation of matrices by Newton-Schulz products, for optimizers that step along the orthogonal factor of an update.
//
//   X = G / (|G|_F + eps); `steps` times: A = X X^T (X^T X for a matrix of more rows than columns), P = b A + c A^2, X <- a X + P X
//   (X P): an odd polynomial of degree five applied to the singular values.
//
// Arithmetic. Operands of the products are FP16 (11 bits, as many as TF32 has, at twice its rate; 8 bits of BF16 would be 5 % off for
// matrices with a few strong directions), sums FP32. The iterate is carried as the sum of two FP16 numbers, X = hi + lo: the product
// takes hi, the linear term a X takes both. With hi alone the rounding of the strong directions, spread over all directions and
// amplified a-fold per step as the weak ones are, is 0.8 % of the result for strong directions 20 times the others (3 % for 200
// times), with the pair 0.02-0.2 %. X is kept times 2^10, which takes its elements (about 1 / sqrt(rows * cols)) out of the range
// where FP16 loses bits.
#include "common.cuh"
#include "tcgen05.cuh"

namespace {
using namespace gdb_t5;

constexpr float NS_UP = 1024.0f, NS_DOWN = 1.0f / 1024.0f;
constexpr int NS_NORM_BLOCKS = 64;   // partial sums of a matrix's squares, at most

// ------------------------------------------------------------------ |G|_F and the first iterate
// Sums of squares are FP64: neither 1e38 nor 1e-38 leaves the range, and the order of the sum does not show.
template <typename T>
__global__ void __launch_bounds__(256)
ns_norm_kernel(const T *__restrict__ g, double *__restrict__ partial, size_t count)
{
    gdb_pdl_sync();
    __shared__ double sh[8];
    const T *m = g + (size_t)blockIdx.y * count;
    double s = 0.0;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (size_t)gridDim.x * blockDim.x) {
        const double v = (double)gdb_io<T>::ld(m, i);
        s += v * v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffU, s, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) s += sh[w];
        partial[(size_t)blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = s;
    }
}
template <typename T>
__global__ void __launch_bounds__(256)
ns_split_kernel(const T *__restrict__ g, const double *__restrict__ partial, int parts, __half *__restrict__ hi, __half *__restrict__ lo, size_t rows, size_t cols, size_t pitch,
                float eps)
{
    gdb_pdl_sync();
    double s = 0.0;
    for (int k = 0; k < parts; ++k) s += __ldg(&partial[(size_t)blockIdx.y * NS_NORM_BLOCKS + k]);
    const double f = (double)NS_UP / (sqrt(s) + (double)eps);
    const T *m = g + (size_t)blockIdx.y * rows * cols;
    __half *h = hi + (size_t)blockIdx.y * rows * pitch, *l = lo + (size_t)blockIdx.y * rows * pitch;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * cols; i += (size_t)gridDim.x * blockDim.x) {
        const size_t r = i / cols, c = i - r * cols;
        const float v = (float)((double)gdb_io<T>::ld(m, i) * f);
        const __half a = __float2half_rn(v);
        h[r * pitch + c] = a;
        l[r * pitch + c] = __float2half_rn(v - __half2float(a));
    }
}

// ------------------------------------------------------------------ products
enum { NS_GRAM, NS_POLY, NS_UPDATE, NS_LAST };

struct ns_epilogue {
    __half *out, *out_lo;            // GRAM / POLY: the symmetric product; UPDATE: the next iterate
    const __half *in, *in_lo;        // POLY: A; UPDATE / LAST: this iterate
    void *final_out;                 // LAST
    size_t out_batch, out_pitch;     // elements
    size_t in_batch, in_pitch;
    float alpha, beta;               // alpha * product + beta * in
};

constexpr int NS_STAGES = 4, NS_BN = 128;
constexpr int NS_STAGE_BYTES = (BM + NS_BN) * BK * 2;
constexpr int NS_SMEM = NS_STAGES * NS_STAGE_BYTES + 256 + 1024;

// One 128 x 128 tile per CTA. GRAM and POLY are symmetric: tiles on and above the diagonal are formed, those above it written twice.
template <bool A_MN, bool B_MN, int MODE, typename TOUT>
__global__ void __launch_bounds__(192, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, ns_epilogue ep, uint32_t M, uint32_t N, uint32_t K, uint32_t tiles_n,
                  int *err_flag)
{
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023U) & ~(uintptr_t)1023U);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + NS_STAGES * NS_STAGE_BYTES);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * NS_STAGES + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t tm, tn;
    if (SYM) {
        // row tm of the upper triangle holds tiles_n - tm tiles
        uint32_t u = blockIdx.x;
        for (tm = 0; u >= tiles_n - tm; ++tm) u -= tiles_n - tm;
        tn = tm + u;
    } else {
        tm = blockIdx.x / tiles_n;
        tn = blockIdx.x - tm * tiles_n;
    }
    const uint32_t m0 = tm * BM, n0 = tn * NS_BN, n_iters = (K + BK - 1) / BK;
    const int z = (int)blockIdx.y;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[NS_STAGES]), accum_bar = smem_u32(&bars[2 * NS_STAGES]);
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS_STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(accum_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)NS_BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    gdb_pdl_sync();

    if (warp == 0) {
        if (lane == 0) {
            for (uint32_t it = 0; it < n_iters; ++it) {
                const uint32_t s = it % NS_STAGES, ph = (it / NS_STAGES) & 1U, bar = full0 + 8 * s;
                if (!mbar_wait(empty0 + 8 * s, ph ^ 1U)) {
                    atomicExch(err_flag, 701);
                    break;
                }
                const uint32_t a_dst = smem_u32(smem + s * NS_STAGE_BYTES), b_dst = a_dst + BM * BK * 2;
                const int k0 = (int)(it * BK);
                mbar_expect_tx(bar, NS_STAGE_BYTES);
                if (A_MN) {
                    tma_load_3d(a_dst, &tma_a, (int)m0, k0, z, bar);
                    tma_load_3d(a_dst + BK * 128, &tma_a, (int)m0 + 64, k0, z, bar);
                } else {
                    tma_load_3d(a_dst, &tma_a, k0, (int)m0, z, bar);
                }
                if (B_MN) {
                    tma_load_3d(b_dst, &tma_b, (int)n0, k0, z, bar);
                    tma_load_3d(b_dst + BK * 128, &tma_b, (int)n0 + 64, k0, z, bar);
                } else {
                    tma_load_3d(b_dst, &tma_b, k0, (int)n0, z, bar);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t IDESC = (1U << 4) | ((A_MN ? 1U : 0U) << 15) | ((B_MN ? 1U : 0U) << 16) | ((uint32_t)(NS_BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            for (uint32_t it = 0; it < n_iters; ++it) {
                const uint32_t s = it % NS_STAGES, ph = (it / NS_STAGES) & 1U;
                if (!mbar_wait(full0 + 8 * s, ph)) {
                    atomicExch(err_flag, 702);
                    break;
                }
                tcgen05_fence_after();
                const uint32_t a_base = smem_u32(smem + s * NS_STAGE_BYTES), b_base = a_base + BM * BK * 2;
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
        const int quad = warp & 3;
        const uint32_t row = m0 + quad * 32 + lane;
        const bool ok = mbar_wait(accum_bar, 0);
        if (!ok && lane == 0) atomicExch(err_flag, 703);
        tcgen05_fence_after();
        if (ok) {
#pragma unroll 1
            for (int cb = 0; cb < NS_BN / 32; ++cb) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(cb * 32), v);
                const uint32_t col0 = n0 + cb * 32;
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    if (row >= M || col0 + j >= N) continue;
                    float f[8];
                    gdb_vec8<__half> a, o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = ep.alpha * __uint_as_float(v[j + e]);
                    if (MODE != NS_GRAM) {
                        const size_t at = (size_t)z * ep.in_batch + (size_t)row * ep.in_pitch + col0 + j;
                        a.raw = *reinterpret_cast<const uint4 *>(ep.in + at);
                        if (MODE == NS_POLY) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] += ep.beta * a.get(e);
                        } else {
                            gdb_vec8<__half> l;
                            l.raw = *reinterpret_cast<const uint4 *>(ep.in_lo + at);
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] += ep.beta * (a.get(e) + l.get(e));
                        }
                    }
                    if (MODE == NS_LAST) {
                        TOUT *dst = reinterpret_cast<TOUT *>(ep.final_out) + (size_t)z * ep.out_batch + (size_t)row * ep.out_pitch + col0 + j;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (col0 + j + e < N) gdb_io<TOUT>::st(dst, e, f[e] * NS_DOWN);
                        }
                        continue;
                    }
                    const size_t at = (size_t)z * ep.out_batch + (size_t)row * ep.out_pitch + col0 + j;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o.set(e, f[e]);
                    *reinterpret_cast<uint4 *>(ep.out + at) = o.raw;
                    if (MODE == NS_UPDATE) {
                        gdb_vec8<__half> l;
#pragma unroll
                        for (int e = 0; e < 8; ++e) l.set(e, f[e] - o.get(e));
                        *reinterpret_cast<uint4 *>(ep.out_lo + at) = l.raw;
                    }
                    if (SYM && tn != tm) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (col0 + j + e < N) ep.out[(size_t)z * ep.out_batch + (size_t)(col0 + j + e) * ep.out_pitch + row] = __ushort_as_half((unsigned short)((&o.raw.x)[e >> 1] >> (16 * (e & 1))));
                        }
                    }
                }
                __syncwarp();   // (the next load from tensor memory is the whole warp's)
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)NS_BN) : "memory");
    }
}

template <bool A_MN, bool B_MN, int MODE, typename TOUT>
gd_status product(gd_backend *be, const CUtensorMap &ma, const CUtensorMap &mb, const ns_epilogue &ep, uint32_t M, uint32_t N, uint32_t K, uint32_t batch)
{
    auto kern = ns_product_kernel<A_MN, B_MN, MODE, TOUT>;
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM);
        if (e != cudaSuccess) return gdb_fail(be, e, "orthogonalize smem attribute");
        ready = true;
    }
    const uint32_t tiles_m = (M + BM - 1) / BM, tiles_n = (N + NS_BN - 1) / NS_BN;
    const uint32_t tiles = MODE == NS_GRAM || MODE == NS_POLY ? tiles_n * (tiles_n + 1) / 2 : tiles_m * tiles_n;
    gdb_launch(kern, dim3(tiles, batch), 192, NS_SMEM, be->stream, ma, mb, ep, M, N, K, tiles_n, be->err_flag);
    return gdb_launched(be, "orthogonalize product");
}

// Where the parts of the scratch lie: the iterate's high halves (two, used in turn), its low halves, A, P, the sums of squares.
struct ns_layout {
    size_t small, pitch, small_pitch;
    size_t hi[2], lo, gram, poly, norm, total;
};
bool ns_plan(const gdb200_orthogonalize_args *a, ns_layout *l)
{
    if (a == NULL || a->rows >= (1U << 24) || a->cols >= (1U << 24) || a->batch > 65535U) return false;
    l->small = a->rows < a->cols ? a->rows : a->cols;
    l->pitch = (a->cols + 7U) & ~(uint64_t)7U;
    l->small_pitch = (l->small + 7U) & ~(size_t)7U;
    if (l->pitch != 0U && a->rows * l->pitch > (SIZE_MAX >> 8) / (a->batch + 1U)) return false;
    const size_t x = (a->batch * a->rows * l->pitch * 2U + 255U) & ~(size_t)255U, s = (a->batch * l->small * l->small_pitch * 2U + 255U) & ~(size_t)255U;
    l->hi[0] = 0U;
    l->hi[1] = x;
    l->lo = 2U * x;
    l->gram = 3U * x;
    l->poly = 3U * x + s;
    l->norm = 3U * x + 2U * s;
    l->total = l->norm + a->batch * NS_NORM_BLOCKS * sizeof(double);
    return true;
}

template <typename T>
gd_status first_iterate(gd_backend *be, const void *g, double *partial, __half *hi, __half *lo, const gdb200_orthogonalize_args *a, size_t pitch)
{
    const size_t count = a->rows * a->cols;
    unsigned parts = (unsigned)((count + 8191U) / 8192U < NS_NORM_BLOCKS ? (count + 8191U) / 8192U : NS_NORM_BLOCKS);
    gdb_launch(ns_norm_kernel<T>, dim3(parts, (unsigned)a->batch), 256, 0, be->stream, (const T *)g, partial, count);
    gd_status st = gdb_launched(be, "orthogonalize norm");
    if (st != GD_OK) return st;
    gdb_launch(ns_split_kernel<T>, dim3(gdb_grid_for(count, 1024, be, 4), (unsigned)a->batch), 256, 0, be->stream, (const T *)g, (const double *)partial, (int)parts, hi, lo,
               (size_t)a->rows, (size_t)a->cols, pitch, a->eps);
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
    if (be == NULL || x == NULL || out == NULL || scratch == NULL || a == NULL || a->steps == 0U || !(a->eps >= 0.0f)) {
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
    const uint32_t rows = (uint32_t)a->rows, cols = (uint32_t)a->cols, m = (uint32_t)l.small, batch = (uint32_t)a->batch;
    const bool tall = rows > cols;
    __half *hi[2] = {(__half *)(sp + l.hi[0]), (__half *)(sp + l.hi[1])}, *lo = (__half *)(sp + l.lo), *gram = (__half *)(sp + l.gram), *poly = (__half *)(sp + l.poly);
    // operand tiles: [k contiguous] boxes of 128 rows, [k strided] boxes of 64 columns
    CUtensorMap xk[2], xm[2], gk, pk;
    bool ok = make_tmap_batched(&gk, GDB_DTYPE_F16, gram, batch, m, m, l.small_pitch * 2U, m * l.small_pitch * 2U, BK, 128) &&
              make_tmap_batched(&pk, GDB_DTYPE_F16, poly, batch, m, m, l.small_pitch * 2U, m * l.small_pitch * 2U, BK, 128);
    for (int i = 0; i < 2; ++i) {
        ok = ok && make_tmap_batched(&xk[i], GDB_DTYPE_F16, hi[i], batch, rows, cols, l.pitch * 2U, rows * l.pitch * 2U, BK, 128) &&
             make_tmap_batched(&xm[i], GDB_DTYPE_F16, hi[i], batch, rows, cols, l.pitch * 2U, rows * l.pitch * 2U, 64, BK);
    }
    if (!ok) {
        return GD_ERR_UNSUPPORTED;
    }
    double *norm = (double *)(sp + l.norm);
    gd_status st = x->dtype == GDB_DTYPE_F16    ? first_iterate<__half>(be, xp, norm, hi[0], lo, a, l.pitch)
                   : x->dtype == GDB_DTYPE_BF16 ? first_iterate<__nv_bfloat16>(be, xp, norm, hi[0], lo, a, l.pitch)
                                                : first_iterate<float>(be, xp, norm, hi[0], lo, a, l.pitch);
    ns_epilogue square = {};
    square.out_batch = square.in_batch = m * l.small_pitch;
    square.out_pitch = square.in_pitch = l.small_pitch;
    for (uint32_t k = 0; k < a->steps && st == GD_OK; ++k) {
        const int cur = (int)(k & 1U);
        ns_epilogue e = square;
        e.out = gram;
        e.alpha = NS_DOWN * NS_DOWN;
        st = tall ? product<true, true, NS_GRAM, __half>(be, xm[cur], xm[cur], e, m, m, rows, batch) : product<false, false, NS_GRAM, __half>(be, xk[cur], xk[cur], e, m, m, cols, batch);
        if (st != GD_OK) break;
        e.in = gram;
        e.out = poly;
        e.alpha = a->c;
        e.beta = a->b;
        st = product<false, false, NS_POLY, __half>(be, gk, gk, e, m, m, m, batch);
        if (st != GD_OK) break;
        e = ns_epilogue();
        e.in = hi[cur];
        e.in_lo = lo;
        e.in_batch = e.out_batch = rows * l.pitch;
        e.in_pitch = e.out_pitch = l.pitch;
        e.alpha = 1.0f;
        e.beta = a->a;
        if (k + 1U < a->steps) {
            e.out = hi[cur ^ 1];
            e.out_lo = lo;
            st = tall ? product<false, false, NS_UPDATE, __half>(be, xk[cur], pk, e, rows, cols, m, batch) : product<false, true, NS_UPDATE, __half>(be, pk, xm[cur], e, rows, cols, m, batch);
        } else {
            e.final_out = op;
            e.out_batch = (size_t)rows * cols;
            e.out_pitch = cols;
#define GO(T) (tall ? product<false, false, NS_LAST, T>(be, xk[cur], pk, e, rows, cols, m, batch) : product<false, true, NS_LAST, T>(be, pk, xm[cur], e, rows, cols, m, batch))
            st = out->dtype == GDB_DTYPE_F16 ? GO(__half) : GO(__nv_bfloat16);
#undef GO
        }
    }
    return st;
}

}  // extern "C"
