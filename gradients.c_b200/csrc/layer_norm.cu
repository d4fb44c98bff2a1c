// Layer norm, forward and backward with the weight's and the bias's gradient.
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), h = (x - mu) r, y = h w + b
//   dx = r (g w - mean(g w) - h mean(g w h)), dw = sum over rows of g h, db = sum over rows of g
//
// HBM-bound: forward reads x and writes y, backward reads x and g and writes dx. A row lies in the registers of a group of TPR
// threads, 16 elements a thread, so that mean and variance are two passes over registers (no cancellation of sums of squares) and
// x is read once. All sums are FP32.
#include "common.cuh"

namespace {

constexpr int LN_EPT = 16;                       // elements of a row that a thread holds
constexpr size_t LN_MAX_COLS = 512 * LN_EPT;     // rows that a group of one block's threads holds

// VE consecutive elements, moved with one access (VE > 1: 16 bytes)
template <typename T, int VE> struct ln_vec;
template <typename T> struct ln_vec<T, 1> {
    static __device__ __forceinline__ void ld(const T *p, float (&f)[1]) { f[0] = gdb_io<T>::ld(p, 0); }
    static __device__ __forceinline__ void st(T *p, const float (&f)[1]) { gdb_io<T>::st(p, 0, f[0]); }
};
template <typename T> struct ln_vec<T, 8> {
    static __device__ __forceinline__ void ld(const T *p, float (&f)[8])
    {
        gdb_vec8<T> v;
        v.raw = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v.get(e);
    }
    static __device__ __forceinline__ void st(T *p, const float (&f)[8])
    {
        gdb_vec8<T> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.set(e, f[e]);
        *reinterpret_cast<uint4 *>(p) = v.raw;
    }
};
template <> struct ln_vec<float, 4> {
    static __device__ __forceinline__ void ld(const float *p, float (&f)[4])
    {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        f[0] = v.x;
        f[1] = v.y;
        f[2] = v.z;
        f[3] = v.w;
    }
    static __device__ __forceinline__ void st(float *p, const float (&f)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};

// Sums over a group of TPR threads of a block. Groups of more than a warp meet at a named barrier of their own; `sh` holds two sets of
// one value pair per warp of the block, used in turn (`flip`), so that one barrier a call is enough.
template <int TPR>
__device__ __forceinline__ float2 ln_group_sum(float2 v, float2 *sh, unsigned flip)
{
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffU, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffU, v.y, o);
    }
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int warp = threadIdx.x >> 5, group = threadIdx.x / TPR;
        float2 *s = sh + flip * 32U;
        if ((threadIdx.x & 31) == 0) s[warp] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(TPR) : "memory");
        v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            v.x += s[group * W + w].x;
            v.y += s[group * W + w].y;
        }
    }
    return v;
}

// One row per group, LN_FWD_THREADS / TPR rows per block. stats (may be NULL): mean and 1 / deviation of every row.
template <typename T, int TPR, int VE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
layer_norm_fwd_kernel(const T *x, const T *__restrict__ w, const T *__restrict__ b, T *out, float2 *__restrict__ stats, size_t rows, unsigned cols, float eps)
{
    gdb_pdl_sync();
    constexpr int NV = LN_EPT / VE, THREADS = TPR > 256 ? TPR : 256;
    __shared__ float2 sh[64];
    const unsigned t = threadIdx.x % TPR;
    const size_t row = (size_t)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
    const bool live = row < rows;   // (groups within a warp stay together through the shuffles)
    const T *xr = x + (live ? row : 0) * cols;
    float f[NV][VE];
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const unsigned c = (t + j * TPR) * VE;
#pragma unroll
        for (int e = 0; e < VE; ++e) f[j][e] = 0.0f;
        if (live && c < cols) ln_vec<T, VE>::ld(xr + c, f[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < VE; ++e) s.x += f[j][e];
    }
    const float inv_cols = 1.0f / (float)cols;
    const float mean = ln_group_sum<TPR>(s, sh, 0).x * inv_cols;
    s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if ((t + j * TPR) * VE < cols) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                f[j][e] -= mean;
                s.x += f[j][e] * f[j][e];
            }
        }
    }
    const float inv = rsqrtf(ln_group_sum<TPR>(s, sh, 1).x * inv_cols + eps);
    if (!live) return;
    if (stats != nullptr && t == 0) stats[row] = make_float2(mean, inv);
    T *orow = out + row * cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const unsigned c = (t + j * TPR) * VE;
        if (c < cols) {
            float wf[VE], bf[VE], o[VE];
            if (w != nullptr) ln_vec<T, VE>::ld(w + c, wf);
            if (b != nullptr) ln_vec<T, VE>::ld(b + c, bf);
#pragma unroll
            for (int e = 0; e < VE; ++e) o[e] = fmaf(f[j][e] * inv, w != nullptr ? wf[e] : 1.0f, b != nullptr ? bf[e] : 0.0f);
            ln_vec<T, VE>::st(orow + c, o);
        }
    }
}

// Rows of more than LN_MAX_COLS elements: a block per row that reads x three times (the second and third time from L2).
template <typename T>
__global__ void __launch_bounds__(512)
layer_norm_fwd_long_kernel(const T *x, const T *__restrict__ w, const T *__restrict__ b, T *out, float2 *__restrict__ stats, size_t rows, size_t cols, float eps)
{
    gdb_pdl_sync();
    __shared__ float sh[33];
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols;
        float s = 0.0f;
        for (size_t c = threadIdx.x; c < cols; c += blockDim.x) s += gdb_io<T>::ld(xr, c);
        const float mean = gdb_block_sum(s, sh) / (float)cols;
        s = 0.0f;
        for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float d = gdb_io<T>::ld(xr, c) - mean;
            s += d * d;
        }
        const float inv = rsqrtf(gdb_block_sum(s, sh) / (float)cols + eps);
        if (stats != nullptr && threadIdx.x == 0) stats[row] = make_float2(mean, inv);
        for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float h = (gdb_io<T>::ld(xr, c) - mean) * inv;
            gdb_io<T>::st(out, row * cols + c, fmaf(h, w != nullptr ? gdb_io<T>::ld(w, c) : 1.0f, b != nullptr ? gdb_io<T>::ld(b, c) : 0.0f));
        }
    }
}

// Input gradient and this block's share of the weight's and the bias's gradient from one pass over x and g. Groups of TPR threads walk
// over the rows; the thread's columns of dw and db stay in its registers, the block's sums go to partial[block, 2, cols].
constexpr int LN_BWD_THREADS = 512;
template <typename T, int TPR, int VE>
__global__ void __launch_bounds__(LN_BWD_THREADS, 1)
layer_norm_bwd_kernel(const T *__restrict__ x, const T *__restrict__ w, const float2 *__restrict__ stats, const T *g, T *dx, bool add_to_dx,
                      float *__restrict__ partial, size_t rows, unsigned cols)
{
    gdb_pdl_sync();
    constexpr int NV = LN_EPT / VE, GROUPS = LN_BWD_THREADS / TPR;
    extern __shared__ float sums[];   // [2, cols]
    __shared__ float2 sh[64];
    const unsigned t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float wf[NV][VE], dw[NV][VE], db[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const unsigned c = (t + j * TPR) * VE;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            wf[j][e] = w != nullptr ? 0.0f : 1.0f;
            dw[j][e] = db[j][e] = 0.0f;
        }
        if (w != nullptr && c < cols) ln_vec<T, VE>::ld(w + c, wf[j]);
    }
    const float inv_cols = 1.0f / (float)cols;
    const size_t stride = (size_t)gridDim.x * GROUPS;
    unsigned flip = 0;
    // (the groups of a warp take the same number of turns)
    for (size_t first = (size_t)blockIdx.x * GROUPS + (TPR < 32 ? group & ~(32U / TPR - 1U) : group); first < rows; first += stride) {
        const size_t row = TPR < 32 ? first + (group & (32U / (TPR < 32 ? TPR : 32) - 1U)) : first;
        const bool live = row < rows;
        const size_t at = (live ? row : 0) * cols;
        float h[NV][VE], gf[NV][VE];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const unsigned c = (t + j * TPR) * VE;
#pragma unroll
            for (int e = 0; e < VE; ++e) h[j][e] = gf[j][e] = 0.0f;
            if (live && c < cols) {
                ln_vec<T, VE>::ld(x + at + c, h[j]);
                ln_vec<T, VE>::ld(g + at + c, gf[j]);
            }
        }
        const float2 st = live ? stats[row] : make_float2(0.0f, 0.0f);
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                h[j][e] = (h[j][e] - st.x) * st.y;
                dw[j][e] += gf[j][e] * h[j][e];
                db[j][e] += gf[j][e];
                gf[j][e] *= wf[j][e];
                s.x += gf[j][e];
                s.y += gf[j][e] * h[j][e];
            }
        }
        s = ln_group_sum<TPR>(s, sh, flip);
        flip ^= 1U;
        const float c1 = s.x * inv_cols, c2 = s.y * inv_cols;
        if (live && dx != nullptr) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const unsigned c = (t + j * TPR) * VE;
                if (c < cols) {
                    float o[VE];
#pragma unroll
                    for (int e = 0; e < VE; ++e) o[e] = __fmul_rn(st.y, gf[j][e] - c1 - h[j][e] * c2);   // (never fused with the addition below)
                    if (add_to_dx) {
                        // round, add, round: the entry without accumulation followed by gd_backend_accumulate
                        float d[VE];
                        ln_vec<T, VE>::ld(dx + at + c, d);
#pragma unroll
                        for (int e = 0; e < VE; ++e) o[e] = d[e] + gdb_io<T>::rnd(o[e]);
                    }
                    ln_vec<T, VE>::st(dx + at + c, o);
                }
            }
        }
    }
    if (partial == nullptr) return;
    // groups in order
    for (unsigned gr = 0; gr < GROUPS; ++gr) {
        if (gr == group) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const unsigned c = (t + j * TPR) * VE;
                if (c < cols) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        sums[c + e] = (gr == 0 ? 0.0f : sums[c + e]) + dw[j][e];
                        sums[cols + c + e] = (gr == 0 ? 0.0f : sums[cols + c + e]) + db[j][e];
                    }
                }
            }
        }
        __syncthreads();
    }
    for (unsigned c = threadIdx.x; c < 2U * cols; c += LN_BWD_THREADS) partial[(size_t)blockIdx.x * 2U * cols + c] = sums[c];
}

// Rows of more than LN_MAX_COLS elements.
template <typename T>
__global__ void __launch_bounds__(512)
layer_norm_bwd_long_kernel(const T *__restrict__ x, const T *__restrict__ w, const float2 *__restrict__ stats, const T *g, T *dx, bool add_to_dx,
                           size_t rows, size_t cols)
{
    gdb_pdl_sync();
    __shared__ float sh[33];
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols, *gr = g + row * cols;
        const float2 st = stats[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float gw = gdb_io<T>::ld(gr, c) * (w != nullptr ? gdb_io<T>::ld(w, c) : 1.0f);
            s1 += gw;
            s2 += gw * ((gdb_io<T>::ld(xr, c) - st.x) * st.y);
        }
        const float c1 = gdb_block_sum(s1, sh) / (float)cols, c2 = gdb_block_sum(s2, sh) / (float)cols;
        for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float gw = gdb_io<T>::ld(gr, c) * (w != nullptr ? gdb_io<T>::ld(w, c) : 1.0f);
            const float o = __fmul_rn(st.y, gw - c1 - (gdb_io<T>::ld(xr, c) - st.x) * st.y * c2);   // (never fused with the addition below)
            gdb_io<T>::st(dx, row * cols + c, add_to_dx ? gdb_io<T>::ld(dx, row * cols + c) + gdb_io<T>::rnd(o) : o);
        }
    }
}
// partial[chunk, 2, cols] for rows [chunk * per, ...): a thread per column
template <typename T>
__global__ void __launch_bounds__(256)
layer_norm_columns_long_kernel(const T *__restrict__ x, const float2 *__restrict__ stats, const T *__restrict__ g, float *__restrict__ partial, size_t rows,
                               size_t cols, size_t per)
{
    gdb_pdl_sync();
    const size_t c = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= cols) return;
    const size_t r1 = min(rows, (size_t)(blockIdx.y + 1U) * per);
    float dw = 0.0f, db = 0.0f;
    for (size_t r = (size_t)blockIdx.y * per; r < r1; ++r) {
        const float2 st = __ldg(&stats[r]);
        const float gf = gdb_io<T>::ld(g, r * cols + c);
        dw += gf * ((gdb_io<T>::ld(x, r * cols + c) - st.x) * st.y);
        db += gf;
    }
    partial[(size_t)blockIdx.y * 2U * cols + c] = dw;
    partial[(size_t)blockIdx.y * 2U * cols + cols + c] = db;
}

// dw[c] and db[c]: the blocks' partial sums in a fixed order (eight threads a column, every eighth block each), rounded once.
template <typename T>
__global__ void __launch_bounds__(256)
layer_norm_merge_kernel(const float *__restrict__ partial, T *__restrict__ dw, T *__restrict__ db, unsigned blocks, size_t cols)
{
    gdb_pdl_sync();
    __shared__ float sh[8][33];
    const unsigned lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const size_t c = (size_t)blockIdx.x * 32U + lane;
    float s = 0.0f;
    if (c < 2U * cols) {
#pragma unroll 4
        for (unsigned k = part; k < blocks; k += 8U) s += __ldcg(&partial[(size_t)k * 2U * cols + c]);
    }
    sh[part][lane] = s;
    __syncthreads();
    if (part == 0 && c < 2U * cols) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += sh[k][lane];
        if (c < cols) {
            if (dw != nullptr) gdb_io<T>::st(dw, c, v);
        } else if (db != nullptr) {
            gdb_io<T>::st(db, c - cols, v);
        }
    }
}

struct ln_call {
    const void *x, *w, *b, *g;
    void *out, *dx, *dw, *db;
    float2 *stats;
    size_t rows, cols;
    float eps;
    bool add_to_dx;
};

// threads of a row: enough for 16 elements each
#define LN_BY_WIDTH(GO, VE)                                                                                                                                   \
    (a.cols <= 8U * LN_EPT      ? GO(8, VE)                                                                                                                   \
     : a.cols <= 16U * LN_EPT   ? GO(16, VE)                                                                                                                  \
     : a.cols <= 32U * LN_EPT   ? GO(32, VE)                                                                                                                  \
     : a.cols <= 64U * LN_EPT   ? GO(64, VE)                                                                                                                  \
     : a.cols <= 128U * LN_EPT  ? GO(128, VE)                                                                                                                 \
     : a.cols <= 256U * LN_EPT  ? GO(256, VE)                                                                                                                 \
                                : GO(512, VE))

template <typename T, int TPR, int VE>
gd_status fwd_go(gd_backend *be, const ln_call &a)
{
    constexpr unsigned THREADS = TPR > 256 ? TPR : 256, PER = THREADS / TPR;
    const size_t blocks = (a.rows + PER - 1U) / PER;
    if (blocks > 0x7fffffffU) return GD_ERR_UNSUPPORTED;
    gdb_launch(layer_norm_fwd_kernel<T, TPR, VE>, (unsigned)blocks, THREADS, 0, be->stream, (const T *)a.x, (const T *)a.w, (const T *)a.b, (T *)a.out, a.stats, a.rows,
               (unsigned)a.cols, a.eps);
    return gdb_launched(be, "layer_norm_forward");
}

template <typename T>
gd_status fwd_typed(gd_backend *be, const ln_call &a)
{
    constexpr int VE = sizeof(T) == 2 ? 8 : 4;
    if (a.cols > LN_MAX_COLS) {
        gdb_launch(layer_norm_fwd_long_kernel<T>, gdb_grid_for(a.rows, 1U, be, 4U), 512, 0, be->stream, (const T *)a.x, (const T *)a.w, (const T *)a.b, (T *)a.out, a.stats, a.rows,
                   a.cols, a.eps);
        return gdb_launched(be, "layer_norm_forward");
    }
    const bool vec = a.cols % VE == 0U && (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.b | (uintptr_t)a.out) % 16U) == 0U;
#define GO(TPR, V) fwd_go<T, TPR, V>(be, a)
    return vec ? LN_BY_WIDTH(GO, VE) : LN_BY_WIDTH(GO, 1);
#undef GO
}

template <typename T, int TPR, int VE>
gd_status bwd_go(gd_backend *be, const ln_call &a, float *partial, unsigned max_blocks, unsigned *blocks)
{
    constexpr unsigned PER = LN_BWD_THREADS / TPR;
    const size_t need = (a.rows + PER - 1U) / PER;
    *blocks = (unsigned)(need < max_blocks ? need : max_blocks);
    const int smem = (int)(2U * a.cols * sizeof(float));
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(layer_norm_bwd_kernel<T, TPR, VE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2U * TPR * LN_EPT * sizeof(float)));
        if (e != cudaSuccess) return gdb_fail(be, e, "layer_norm_backward smem attribute");
        ready = true;
    }
    gdb_launch(layer_norm_bwd_kernel<T, TPR, VE>, *blocks, LN_BWD_THREADS, smem, be->stream, (const T *)a.x, (const T *)a.w, (const float2 *)a.stats, (const T *)a.g, (T *)a.dx,
               a.add_to_dx, partial, a.rows, (unsigned)a.cols);
    return gdb_launched(be, "layer_norm_backward");
}

template <typename T>
gd_status bwd_typed(gd_backend *be, const ln_call &a)
{
    constexpr int VE = sizeof(T) == 2 ? 8 : 4;
    const bool sums = a.dw != nullptr || a.db != nullptr;
    float *partial = sums ? reinterpret_cast<float *>(be->ws) : nullptr;
    const size_t fit = be->ws_bytes / (2U * a.cols * sizeof(float));   // blocks whose partial sums the workspace holds
    if (sums && fit == 0U) return GD_ERR_UNSUPPORTED;
    unsigned blocks = 0;
    gd_status st;
    if (a.cols > LN_MAX_COLS) {
        if (a.dx != nullptr) {
            gdb_launch(layer_norm_bwd_long_kernel<T>, gdb_grid_for(a.rows, 1U, be, 4U), 512, 0, be->stream, (const T *)a.x, (const T *)a.w, (const float2 *)a.stats, (const T *)a.g,
                       (T *)a.dx, a.add_to_dx, a.rows, a.cols);
            st = gdb_launched(be, "layer_norm_backward");
            if (st != GD_OK || !sums) return st;
        }
        const size_t col_blocks = (a.cols + 255U) / 256U;
        size_t chunks = ((size_t)be->sm_count * 8U + col_blocks - 1U) / col_blocks;
        if (chunks > fit) chunks = fit;
        if (chunks > a.rows) chunks = a.rows;
        if (col_blocks > 0x7fffffffU) return GD_ERR_UNSUPPORTED;
        const size_t per = (a.rows + chunks - 1U) / chunks;
        blocks = (unsigned)((a.rows + per - 1U) / per);
        gdb_launch(layer_norm_columns_long_kernel<T>, dim3((unsigned)col_blocks, blocks), 256, 0, be->stream, (const T *)a.x, (const float2 *)a.stats, (const T *)a.g, partial,
                   a.rows, a.cols, per);
        st = gdb_launched(be, "layer_norm_backward columns");
    } else {
        const unsigned most = (unsigned)(!sums || fit > (size_t)be->sm_count ? (size_t)be->sm_count : fit);
        const bool vec = a.cols % VE == 0U && (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.g | (uintptr_t)a.dx) % 16U) == 0U;
#define GO(TPR, V) bwd_go<T, TPR, V>(be, a, partial, most, &blocks)
        st = vec ? LN_BY_WIDTH(GO, VE) : LN_BY_WIDTH(GO, 1);
#undef GO
    }
    if (st != GD_OK || !sums) return st;
    gdb_launch(layer_norm_merge_kernel<T>, (unsigned)((2U * a.cols + 31U) / 32U), 256, 0, be->stream, (const float *)partial, (T *)a.dw, (T *)a.db, blocks, a.cols);
    return gdb_launched(be, "layer_norm_backward merge");
}

// pointer of an optional contiguous tensor of `count` elements; false where it is given and does not fit
bool ln_ptr(const gd_backend_tensor_view *v, uint32_t dtype, size_t count, void **p)
{
    *p = NULL;
    if (v == NULL) return true;
    if (v->count != count) return false;
    *p = gdb_tv_ptr(v, dtype);
    return *p != NULL;
}

bool ln_args_ok(const gdb200_layer_norm_args *a)
{
    return a != NULL && a->cols > 0U && a->rows <= SIZE_MAX / 4U / a->cols && a->eps >= 0.0f;
}

}  // namespace

extern "C" {

gd_status gdb200_layer_norm_forward(gd_backend *be, const gd_backend_tensor_view *x, const gd_backend_tensor_view *weight, const gd_backend_tensor_view *bias,
                                    const gd_backend_tensor_view *out, const gd_backend_tensor_view *stats, const gdb200_layer_norm_args *args)
{
    if (be == NULL || x == NULL || out == NULL || !ln_args_ok(args)) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (!gdb_is_float_dtype(x->dtype)) {
        return GD_ERR_UNSUPPORTED;
    }
    const size_t n = args->rows * args->cols;
    void *xp, *wp, *bp, *op, *sp;
    if (!ln_ptr(x, x->dtype, n, &xp) || !ln_ptr(weight, x->dtype, args->cols, &wp) || !ln_ptr(bias, x->dtype, args->cols, &bp) || !ln_ptr(out, x->dtype, n, &op) ||
        !ln_ptr(stats, GDB_DTYPE_F32, 2U * args->rows, &sp) || ((uintptr_t)sp % 8U) != 0U) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (args->rows == 0U) {
        return GD_OK;
    }
    ln_call a = {};
    a.x = xp;
    a.w = wp;
    a.b = bp;
    a.out = op;
    a.stats = (float2 *)sp;
    a.rows = args->rows;
    a.cols = args->cols;
    a.eps = args->eps;
    return x->dtype == GDB_DTYPE_F16 ? fwd_typed<__half>(be, a) : (x->dtype == GDB_DTYPE_BF16 ? fwd_typed<__nv_bfloat16>(be, a) : fwd_typed<float>(be, a));
}

gd_status gdb200_layer_norm_backward(gd_backend *be, const gd_backend_tensor_view *x, const gd_backend_tensor_view *weight, const gd_backend_tensor_view *stats,
                                     const gd_backend_tensor_view *grad_out, const gd_backend_tensor_view *grad_x, int32_t accumulate,
                                     const gd_backend_tensor_view *grad_weight, const gd_backend_tensor_view *grad_bias, const gdb200_layer_norm_args *args)
{
    if (be == NULL || x == NULL || stats == NULL || grad_out == NULL || !ln_args_ok(args) || (grad_x == NULL && grad_weight == NULL && grad_bias == NULL)) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (!gdb_is_float_dtype(x->dtype)) {
        return GD_ERR_UNSUPPORTED;
    }
    const size_t n = args->rows * args->cols;
    void *xp, *wp, *sp, *gp, *dxp, *dwp, *dbp;
    if (!ln_ptr(x, x->dtype, n, &xp) || !ln_ptr(weight, x->dtype, args->cols, &wp) || !ln_ptr(stats, GDB_DTYPE_F32, 2U * args->rows, &sp) ||
        !ln_ptr(grad_out, x->dtype, n, &gp) || !ln_ptr(grad_x, x->dtype, n, &dxp) || !ln_ptr(grad_weight, x->dtype, args->cols, &dwp) ||
        !ln_ptr(grad_bias, x->dtype, args->cols, &dbp) || ((uintptr_t)sp % 8U) != 0U) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (args->rows == 0U) {
        // an empty sum
        const size_t bytes = args->cols * gdb_dtype_size(x->dtype);
        for (void *p : {dwp, dbp}) {
            if (p == NULL) continue;
            const cudaError_t e = cudaMemsetAsync(p, 0, bytes, be->stream);
            be->launches += 1U;
            if (e != cudaSuccess) return gdb_fail(be, e, "layer_norm_backward zero");
        }
        return GD_OK;
    }
    ln_call a = {};
    a.x = xp;
    a.w = wp;
    a.g = gp;
    a.dx = dxp;
    a.dw = dwp;
    a.db = dbp;
    a.stats = (float2 *)sp;
    a.rows = args->rows;
    a.cols = args->cols;
    a.add_to_dx = accumulate != 0;
    return x->dtype == GDB_DTYPE_F16 ? bwd_typed<__half>(be, a) : (x->dtype == GDB_DTYPE_BF16 ? bwd_typed<__nv_bfloat16>(be, a) : bwd_typed<float>(be, a));
}

}  // extern "C"
