// Layer norm, forward and backward with the weight's and the bias's gradient.
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), h = (x - mu) r, y = h w + b
//   dx = r (g w - mean(g w) - h mean(g w h)), dw = sum over rows of g h, db = sum over rows of g
//
// HBM-bound: forward reads x and writes y, backward reads x and g and writes dx. A row lies in the registers of a group of TPR
// threads, 16 elements a thread, so that mean and variance are two passes over registers (no cancellation of sums of squares) and
// x is read once. All sums are FP32. 16384 x 2048 BF16: forward 23.4 us (5.7 TB/s), backward 41 (4.9); 18432 x 512 FP16 8.1 and 13.5.
#include "common.cuh"
#include "tcgen05.cuh"

namespace {
using namespace gdb_t5;

constexpr int LN_EPT = 16;                       // elements of a row that a thread holds
constexpr size_t LN_MAX_COLS = 512 * LN_EPT;     // rows that a group of one block's threads holds

// VE consecutive elements, stored with one access (VE > 1: 16 bytes)
template <typename T, int VE> struct ln_vec;
template <typename T> struct ln_vec<T, 1> {
    static __device__ __forceinline__ void st(T *p, const float (&f)[1]) { gdb_io<T>::st(p, 0, f[0]); }
};
// (two 16-bit elements a conversion)
template <typename T> __device__ __forceinline__ float2 ln_two(uint32_t w);
template <> __device__ __forceinline__ float2 ln_two<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
template <> __device__ __forceinline__ float2 ln_two<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000U)); }
template <typename T> struct ln_vec<T, 8> {
    static __device__ __forceinline__ void st(T *p, const float (&f)[8])
    {
        *reinterpret_cast<uint4 *>(p) = make_uint4(half_pack<T>::pack(f[0], f[1]), half_pack<T>::pack(f[2], f[3]), half_pack<T>::pack(f[4], f[5]), half_pack<T>::pack(f[6], f[7]));
    }
};
template <> struct ln_vec<float, 4> {
    static __device__ __forceinline__ void st(float *p, const float (&f)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};

// Sums of K value pairs over a group of TPR threads of a block. Groups of more than a warp meet at a named barrier of their own; `sh` holds
// two sets of K pairs per warp of the block (at most 16), used in turn (`flip`), so that one barrier a call is enough.
template <int TPR, int K>
__device__ __forceinline__ void ln_group_sums(float2 (&v)[K], float2 *sh, unsigned flip)
{
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int r = 0; r < K; ++r) {
            v[r].x += __shfl_xor_sync(0xffffffffU, v[r].x, o);
            v[r].y += __shfl_xor_sync(0xffffffffU, v[r].y, o);
        }
    }
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int warp = threadIdx.x >> 5, group = threadIdx.x / TPR;
        float2 *s = sh + flip * (16U * K);
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int r = 0; r < K; ++r) s[warp * K + r] = v[r];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(TPR) : "memory");
#pragma unroll
        for (int r = 0; r < K; ++r) {
            v[r] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                v[r].x += s[(group * W + w) * K + r].x;
                v[r].y += s[(group * W + w) * K + r].y;
            }
        }
    }
}
template <int TPR>
__device__ __forceinline__ float2 ln_group_sum(float2 v, float2 *sh, unsigned flip)
{
    float2 one[1] = {v};
    ln_group_sums<TPR, 1>(one, sh, flip);
    return one[0];
}

// A thread's EPT elements of a row in pairs (sm_100 multiplies and adds two FP32 numbers an instruction): accesses of VE elements, TPR
// accesses apart.
template <typename T, int VE, int TPR, int EPT = LN_EPT> struct ln_pairs {
    f32x2 v[EPT / 2];
    // Rows fill more than half of a group's places (LN_BY_WIDTH), so the first half needs no test.
    static __host__ __device__ constexpr bool inside(int j) { return TPR > 8 && 2 * (j + 1) * VE <= EPT; }
    // a row's elements as they lie in memory, to be taken apart later
    struct raw {
        uint4 v[VE > 1 ? EPT / VE : 1];
        float f[VE > 1 ? 1 : EPT];
        __device__ __forceinline__ void load(const T *p, unsigned t, unsigned cols)
        {
#pragma unroll
            for (int j = 0; j < EPT / VE; ++j) {
                const unsigned c = (t + j * TPR) * VE;
                if (VE > 1) {
                    v[VE > 1 ? j : 0] = make_uint4(0U, 0U, 0U, 0U);
                    if (inside(j) || c < cols) v[VE > 1 ? j : 0] = *reinterpret_cast<const uint4 *>(p + c);
                } else {
                    f[VE > 1 ? 0 : j] = 0.0f;
                    if (inside(j) || c < cols) f[VE > 1 ? 0 : j] = gdb_io<T>::ld(p, c);
                }
            }
        }
    };
    __device__ __forceinline__ void take(const raw &r)
    {
        if constexpr (VE > 1) {
#pragma unroll
            for (int j = 0; j < EPT / VE; ++j) {
                const uint32_t w[4] = {r.v[j].x, r.v[j].y, r.v[j].z, r.v[j].w};
#pragma unroll
                for (int k = 0; k < VE / 2; ++k) {
                    if constexpr (sizeof(T) == 2) {
                        const float2 a = ln_two<T>(w[k]);
                        v[j * (VE / 2) + k] = f2_make(a.x, a.y);
                    } else {
                        v[j * (VE / 2) + k] = f2_make(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
                    }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < EPT / 2; ++k) v[k] = f2_make(r.f[2 * k], r.f[2 * k + 1]);
        }
    }
    __device__ __forceinline__ void fill(float x)
    {
#pragma unroll
        for (int k = 0; k < EPT / 2; ++k) v[k] = f2_make(x, x);
    }
    __device__ __forceinline__ void load(const T *p, unsigned t, unsigned cols)
    {
        raw r;
        r.load(p, t, cols);
        take(r);
    }
    // adds to the elements inside the row
    __device__ __forceinline__ void center(f32x2 by, unsigned t, unsigned cols)
    {
#pragma unroll
        for (int k = 0; k < EPT / 2; ++k) {
            const f32x2 d = f2_add(v[k], by);
            const int j = 2 * k / VE;
            if (VE > 1) {
                if (inside(j) || (t + j * TPR) * VE < cols) v[k] = d;
            } else if (inside(j + 1)) {
                v[k] = d;
            } else {
                float lo, hi, l0, h0;
                f2_split(d, lo, hi);
                f2_split(v[k], l0, h0);
                v[k] = f2_make(t + j * TPR < cols ? lo : l0, t + (j + 1) * TPR < cols ? hi : h0);
            }
        }
    }
    __device__ __forceinline__ void store(T *p, unsigned t, unsigned cols) const
    {
        float f[EPT];
#pragma unroll
        for (int k = 0; k < EPT / 2; ++k) f2_split(v[k], f[2 * k], f[2 * k + 1]);
#pragma unroll
        for (int j = 0; j < EPT / VE; ++j) {
            const unsigned c = (t + j * TPR) * VE;
            if (inside(j) || c < cols) ln_vec<T, VE>::st(p + c, *reinterpret_cast<const float(*)[VE]>(f + j * VE));
        }
    }
};
__device__ __forceinline__ float2 ln_halves(f32x2 s)
{
    float lo, hi;
    f2_split(s, lo, hi);
    return make_float2(lo + hi, 0.0f);
}

// A group walks over rows with the next one on its way; weight and bias stay in registers. stats (may be NULL): mean and 1 / deviation of
// every row.
template <typename T, int TPR, int VE, int EPT>
__device__ __forceinline__ void ln_forward_row(ln_pairs<T, VE, TPR, EPT> &f, const ln_pairs<T, VE, TPR, EPT> &wf, const ln_pairs<T, VE, TPR, EPT> &bf, T *po, float2 *stats, bool live,
                                               unsigned t, unsigned cols, float inv_cols, float eps, float2 *sh)
{
    f32x2 s2 = f2_make(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < EPT / 2; ++k) s2 = f2_add(s2, f.v[k]);
    const float mean = ln_group_sum<TPR>(ln_halves(s2), sh, 0).x * inv_cols;
    f.center(f2_make(-mean, -mean), t, cols);
    s2 = f2_make(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < EPT / 2; ++k) s2 = f2_fma(f.v[k], f.v[k], s2);
    const float inv = rsqrtf(ln_group_sum<TPR>(ln_halves(s2), sh, 1).x * inv_cols + eps);
    if (!live) return;
    if (stats != nullptr && t == 0) *stats = make_float2(mean, inv);
    const f32x2 inv2 = f2_make(inv, inv);
#pragma unroll
    for (int k = 0; k < EPT / 2; ++k) f.v[k] = f2_fma(f2_mul(f.v[k], inv2), wf.v[k], bf.v[k]);
    f.store(po, t, cols);
}
constexpr int LN_AHEAD = 3;                      // rows of a group on their way
__host__ __device__ constexpr int ln_fwd_threads(int tpr) { return tpr > 256 ? tpr : 256; }
// (blocks on an SM, as the registers allow)
__host__ __device__ constexpr int ln_fwd_blocks(int tpr, int ve) { return tpr > 256 ? 1 : (ve > 1 ? 3 : 2); }
template <typename T, int VE> __host__ __device__ constexpr size_t ln_fwd_smem(int tpr) { return VE > 1 ? (size_t)LN_AHEAD * (LN_EPT / VE) * ln_fwd_threads(tpr) * 16U : 0U; }
template <typename T, int TPR, int VE>
__global__ void __launch_bounds__(ln_fwd_threads(TPR), ln_fwd_blocks(TPR, VE))
layer_norm_fwd_kernel(const T *x, const T *__restrict__ w, const T *__restrict__ b, T *out, float2 *__restrict__ stats, size_t rows, unsigned cols, float eps)
{
    gdb_pdl_sync();
    constexpr int THREADS = ln_fwd_threads(TPR), PIECES = LN_EPT / VE;
    constexpr unsigned TOGETHER = TPR < 32 ? 32 / TPR : 1;   // groups of a warp: they take the same number of turns
    __shared__ float2 sh[64];
    extern __shared__ uint4 ahead[];     // [LN_AHEAD, PIECES, THREADS]: a thread copies and reads its own places only
    const unsigned t = threadIdx.x % TPR, group = threadIdx.x / TPR, mine = group % TOGETHER;
    const size_t stride = (size_t)gridDim.x * (THREADS / TPR);
    typedef ln_pairs<T, VE, TPR> pairs;
    size_t first = (size_t)blockIdx.x * (THREADS / TPR) + group - mine;
    typename pairs::raw next;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ahead + threadIdx.x);
    const auto fetch = [&](size_t row, unsigned slot) {
        const T *p = x + row * cols;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const unsigned c = (t + j * TPR) * VE, bytes = pairs::inside(j) || c < cols ? 16U : 0U;   // (the rest of the 16 bytes is zeros)
            if (row < rows) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + (slot * PIECES + j) * (THREADS * 16U)), "l"(bytes != 0U ? p + c : p), "r"(bytes) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (VE > 1) {
#pragma unroll
        for (unsigned k = 0; k < LN_AHEAD; ++k) fetch(first + mine + k * stride, k);
    } else {
        next.load(x + (first + mine < rows ? first + mine : 0) * cols, t, cols);
    }
    pairs wf, bf;
    if (w != nullptr) wf.load(w, t, cols); else wf.fill(1.0f);
    if (b != nullptr) bf.load(b, t, cols); else bf.fill(0.0f);
    const float inv_cols = 1.0f / (float)cols;
    unsigned slot = 0;
    for (; first < rows; first += stride) {
        const size_t row = first + mine;
        pairs f;
        if constexpr (VE > 1) {
            asm volatile("cp.async.wait_group %0;" ::"n"(LN_AHEAD - 1) : "memory");
#pragma unroll
            for (int j = 0; j < PIECES; ++j) next.v[j] = ahead[(slot * PIECES + j) * THREADS + threadIdx.x];
        }
        f.take(next);
        if constexpr (VE == 1) {
            if (first + stride < rows) next.load(x + (row + stride < rows ? row + stride : 0) * cols, t, cols);
        }
        ln_forward_row(f, wf, bf, out + row * cols, stats == nullptr ? nullptr : stats + row, row < rows, t, cols, inv_cols, eps, sh);
        if constexpr (VE > 1) {
            fetch(row + LN_AHEAD * stride, slot);   // (the row that lay there is in registers and behind two exchanges)
            slot = slot + 1U < LN_AHEAD ? slot + 1U : 0U;
        }
    }
    if constexpr (VE > 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
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

// a thread's sums of g h and of g over the rows, for its columns
template <int EPT> struct ln_sums {
    f32x2 dw[EPT / 2], db[EPT / 2];
    __device__ __forceinline__ ln_sums()
    {
#pragma unroll
        for (int k = 0; k < EPT / 2; ++k) dw[k] = db[k] = f2_make(0.0f, 0.0f);
    }
    // to[0, c] and to[1, c] (float4 accesses where VE allows them: to is 16-byte aligned then, and cols a multiple of 4)
    template <int VE, int TPR> __device__ __forceinline__ void store(float *to, unsigned t, unsigned cols) const
    {
        constexpr int A = VE > 1 ? 4 : 1;
#pragma unroll
        for (int q = 0; q < EPT; q += A) {
            const unsigned c = (t + (q / VE) * TPR) * VE + q % VE;
            if (c >= cols) continue;
            float a[2], b[2], u[2], v[2];
            f2_split(dw[q / 2], a[0], a[1]);
            f2_split(db[q / 2], u[0], u[1]);
            if (A == 4) {
                f2_split(dw[(q / 2 + 1) % (EPT / 2)], b[0], b[1]);
                f2_split(db[(q / 2 + 1) % (EPT / 2)], v[0], v[1]);
                *reinterpret_cast<float4 *>(to + c) = make_float4(a[0], a[1], b[0], b[1]);
                *reinterpret_cast<float4 *>(to + cols + c) = make_float4(u[0], u[1], v[0], v[1]);
            } else {
                to[c] = a[q % 2];
                to[cols + c] = u[q % 2];
            }
        }
    }
};
// K rows backward, their sums exchanged together; dead rows go along (shuffles and barriers are the whole warp's). The elements are read
// again behind the exchange, so that K rows are on their way without 32 registers each: one row at a time left 16 warps waiting for
// shuffles (18432 x 512 FP16 17.8 us, of which the memory's 11). px, pg, pd (the old gradient), po (may be px or pg): first row, the others
// `step` elements on.
template <typename T, int VE, int TPR, int EPT, int K>
__device__ __forceinline__ void ln_backward_rows(const T *px, const T *pg, const T *pd, T *po, size_t step, const bool (&live)[K], bool add, const float2 (&st)[K],
                                                 const ln_pairs<T, VE, TPR, EPT> &wf, ln_sums<EPT> &sums, float inv_cols, unsigned t, unsigned cols, float2 *sh, unsigned &flip)
{
    float2 s[K];
#pragma unroll
    for (int r = 0; r < K; ++r) {
        s[r] = make_float2(0.0f, 0.0f);
        if (!live[r]) continue;
        ln_pairs<T, VE, TPR, EPT> h, g;
        h.load(px + r * step, t, cols);
        g.load(pg + r * step, t, cols);
        const f32x2 mean2 = f2_make(-st[r].x, -st[r].x), inv2 = f2_make(st[r].y, st[r].y);
        f32x2 s1 = f2_make(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int k = 0; k < EPT / 2; ++k) {
            // (outside the row g is zero, and h whatever the mean makes of zero)
            const f32x2 hk = f2_mul(f2_add(h.v[k], mean2), inv2), gw = f2_mul(g.v[k], wf.v[k]);
            sums.dw[k] = f2_fma(g.v[k], hk, sums.dw[k]);
            sums.db[k] = f2_add(sums.db[k], g.v[k]);
            s1 = f2_add(s1, gw);
            s2 = f2_fma(gw, hk, s2);
        }
        s[r] = make_float2(ln_halves(s1).x, ln_halves(s2).x);
    }
    ln_group_sums<TPR, K>(s, sh, flip);
    flip ^= 1U;
    if (po == nullptr) return;
#pragma unroll
    for (int r = 0; r < K; ++r) {
        if (!live[r]) continue;
        ln_pairs<T, VE, TPR, EPT> h, g;
        h.load(px + r * step, t, cols);
        g.load(pg + r * step, t, cols);
        const f32x2 mean2 = f2_make(-st[r].x, -st[r].x), inv2 = f2_make(st[r].y, st[r].y);
        const f32x2 c1 = f2_make(-s[r].x * inv_cols, -s[r].x * inv_cols), c2 = f2_make(-s[r].y * inv_cols, -s[r].y * inv_cols);
#pragma unroll
        for (int k = 0; k < EPT / 2; ++k) {
            const f32x2 hk = f2_mul(f2_add(h.v[k], mean2), inv2);
            g.v[k] = f2_mul(inv2, f2_fma(hk, c2, f2_fma(g.v[k], wf.v[k], c1)));
        }
        if (add) {
            // round, add, round: the entry without accumulation followed by gd_backend_accumulate
            h.load(pd + r * step, t, cols);
#pragma unroll
            for (int k = 0; k < EPT / 2; ++k) {
                float a, b;
                f2_split(g.v[k], a, b);
                g.v[k] = f2_add(h.v[k], f2_make(gdb_io<T>::rnd(a), gdb_io<T>::rnd(b)));
            }
        }
        g.store(po + r * step, t, cols);
    }
}

// ---- rows streamed through shared memory: as many bytes on their way as HBM wants, whatever the registers hold ----
// One block per SM walks over tiles of R rows. Bulk copies bring them into a ring, 16 warps work on them, a group of TPR threads per row as
// in the kernel above, and store the result themselves (written into the ring and copied away from there, a stage came free later:
// backward 18432 x 512 FP16 15.2 instead of 13.6 us, 16384 x 2048 BF16 44.0 instead of 41.0, 4099 x 1003 FP32 12.6 instead of 11.8).
// Tiles begin on 16 bytes whatever the width is (R is chosen so), so odd rows stream as even ones do: only the reads from shared memory
// are narrower. A last tile whose bytes are no multiple of 16 is worked on in global memory. The warp that finishes a tile issues the next
// copies into its stage (warps for that alone would leave 96 registers a thread for sums that need 110; one fixed warp among the 16 is
// waited for by all).
constexpr int LN_WARPS = 16, LN_THREADS = LN_WARPS * 32, LN_MAX_STAGES = 8;
constexpr size_t LN_RING_BYTES = 208U * 1024U;

struct ln_stream {
    const void *x, *g, *w, *b;   // g: backward only
    void *out;                   // y, or dx
    float2 *stats;               // written forward (may be NULL), read backward
    float *partial;              // backward: [blocks, 2, cols], or NULL
    size_t rows;
    unsigned cols, tile_rows, tile_bytes, stages;
    float eps;
};

// BWD: 0 forward, 1 backward, 2 backward into a gradient that is there. Streams: x, and g, and the old dx.
template <typename T, int TPR, int VE, int EPT, int BWD>
__global__ void __launch_bounds__(LN_THREADS, 1)
layer_norm_stream_kernel(const ln_stream a, int *err_flag)
{
    constexpr int GROUPS = LN_THREADS / TPR, STREAMS = BWD + 1;
    extern __shared__ __align__(128) unsigned char ring[];   // [stages][streams][tile_bytes], rounded up to 128
    __shared__ __align__(8) uint64_t bars[LN_MAX_STAGES];
    __shared__ unsigned arrived[LN_MAX_STAGES];   // warps that are done with the stage's tile
    __shared__ float2 sh[64];
    const unsigned stages = a.stages, cols = a.cols;
    const uint32_t full0 = smem_u32(bars);
    const size_t slot_bytes = (a.tile_bytes + 127U) & ~127U, stage_bytes = slot_bytes * STREAMS;
    const size_t tiles = (a.rows + a.tile_rows - 1U) / a.tile_rows;
    if (threadIdx.x == 0) {
        for (unsigned s = 0; s < stages; ++s) {
            mbar_init(full0 + 8U * s, 1);
            arrived[s] = 0U;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    gdb_pdl_sync();
    const T *x = reinterpret_cast<const T *>(a.x), *g = reinterpret_cast<const T *>(a.g), *w = reinterpret_cast<const T *>(a.w), *b = reinterpret_cast<const T *>(a.b);
    T *out = reinterpret_cast<T *>(a.out);
    // bytes of a tile that go by bulk copies: all or none
    auto bulk_bytes = [&](size_t tile) {
        const size_t left = a.rows - tile * a.tile_rows, bytes = (left < a.tile_rows ? left : a.tile_rows) * cols * sizeof(T);
        return bytes % 16U == 0U ? (unsigned)bytes : 0U;
    };
    auto fetch = [&](size_t tile, unsigned s) {
        const unsigned bytes = tile < tiles ? bulk_bytes(tile) : 0U;
        if (bytes == 0U) return;
        const size_t at = tile * a.tile_rows * cols;
        const uint32_t dst = smem_u32(ring + s * stage_bytes), bar = full0 + 8U * s;
        mbar_expect_tx(bar, STREAMS * bytes);
        auto copy = [&](int k, const void *src) {
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst + (uint32_t)(k * slot_bytes)), "l"(src), "r"(bytes),
                         "r"(bar)
                         : "memory");
        };
        copy(0, x + at);
        if (BWD >= 1) copy(1, g + at);
        if (BWD == 2) copy(2, out + at);
    };
    if (threadIdx.x == 0) {
        for (unsigned k = 0; k < stages; ++k) fetch(blockIdx.x + (size_t)k * gridDim.x, k);
    }
    const unsigned t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    ln_pairs<T, VE, TPR, EPT> wf, bf;
    if (w != nullptr) wf.load(w, t, cols); else wf.fill(1.0f);
    if (!BWD && b != nullptr) bf.load(b, t, cols); else bf.fill(0.0f);
    ln_sums<EPT> sums2;
    const float inv_cols = 1.0f / (float)cols;
    unsigned flip = 0;
    float2 ahead[2];   // statistics of the group's next two rows
    auto look_ahead = [&](size_t row) {
#pragma unroll
        for (int k = 0; k < 2; ++k) ahead[k] = row + k * GROUPS < a.rows ? __ldg(&a.stats[row + k * GROUPS]) : make_float2(0.0f, 0.0f);
    };
    if (BWD) look_ahead((size_t)blockIdx.x * a.tile_rows + group);
    // rows of a tile (or, behind the last full one, of memory), two at a time backward: first row, rows there are
    auto work = [&](size_t row0, unsigned here, const T *px, const T *pg, const T *pd, T *po) {
        if (BWD) {
            for (unsigned r = group; r < a.tile_rows; r += 2U * GROUPS) {
                const bool live[2] = {r < here, r + GROUPS < here};
                const float2 st[2] = {ahead[0], ahead[1]};
                const bool more = r + 2U * GROUPS < a.tile_rows;
                look_ahead(more ? row0 + r + 2U * GROUPS : row0 + (size_t)gridDim.x * a.tile_rows + group);
                const size_t at = (size_t)r * cols;
                ln_backward_rows<T, VE, TPR, EPT, 2>(px + at, pg + at, pd + at, po == nullptr ? nullptr : po + at, (size_t)GROUPS * cols, live, BWD == 2, st, wf, sums2, inv_cols, t,
                                                     cols, sh, flip);
            }
        } else {
            for (unsigned r = group; r < a.tile_rows; r += GROUPS) {
                ln_pairs<T, VE, TPR, EPT> f;
                if (r < here) f.load(px + (size_t)r * cols, t, cols); else f.fill(0.0f);
                ln_forward_row(f, wf, bf, po + (size_t)r * cols, a.stats == nullptr ? nullptr : a.stats + row0 + r, r < here, t, cols, inv_cols, a.eps, sh);
            }
        }
    };
    unsigned s = 0, ph = 0;
    bool ok = true;
    for (size_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const size_t row0 = tile * a.tile_rows, left = a.rows - row0;
        const unsigned here = left < a.tile_rows ? (unsigned)left : a.tile_rows;
        if (bulk_bytes(tile) == 0U) {
            const size_t at = row0 * cols;
            work(row0, here, x + at, g + at, out + at, out == nullptr ? nullptr : out + at);
            break;
        }
        // (a wait that gives up is not waited for again, and the walk goes on: the groups' barriers stay complete)
        if (ok && !mbar_wait(full0 + 8U * s, ph)) {
            ok = false;
            atomicExch(err_flag, 603);
        }
        __syncwarp();
        T *sx = reinterpret_cast<T *>(ring + s * stage_bytes), *sg = reinterpret_cast<T *>(ring + s * stage_bytes + (BWD >= 1 ? slot_bytes : 0U)),
          *sd = reinterpret_cast<T *>(ring + s * stage_bytes + (BWD == 2 ? 2U * slot_bytes : 0U));
        work(row0, here, sx, sg, sd, out == nullptr ? nullptr : out + row0 * cols);
        // the warp that finishes the tile fetches the next one for its stage
        fence_proxy_async_smem();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            __threadfence_block();
            if (atomicAdd(&arrived[s], 1U) == LN_WARPS - 1U) {
                arrived[s] = 0U;
                __threadfence_block();
                fetch(tile + (size_t)stages * gridDim.x, s);
            }
        }
        if (++s == stages) {
            s = 0;
            ph ^= 1U;
        }
    }
    if (BWD && a.partial != nullptr) {
        // the groups' sums through the ring (64 KB), added in order
        __syncthreads();
        float *sums = reinterpret_cast<float *>(ring);
        sums2.template store<VE, TPR>(sums + (size_t)group * 2U * cols, t, cols);
        __syncthreads();
        for (unsigned c = threadIdx.x; c < 2U * cols; c += LN_THREADS) {
            float v = 0.0f;
#pragma unroll 8
            for (unsigned k = 0; k < GROUPS; ++k) v += sums[(size_t)k * 2U * cols + c];
            a.partial[(size_t)blockIdx.x * 2U * cols + c] = v;
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
    constexpr int GROUPS = LN_BWD_THREADS / TPR;
    extern __shared__ __align__(16) float sums[];   // [groups, 2, cols]
    __shared__ float2 sh[64];
    const unsigned t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    ln_pairs<T, VE, TPR> wf;
    if (w != nullptr) wf.load(w, t, cols); else wf.fill(1.0f);
    ln_sums<LN_EPT> sums2;
    const float inv_cols = 1.0f / (float)cols;
    const size_t stride = (size_t)gridDim.x * GROUPS;
    unsigned flip = 0;
    // (the groups of a warp take the same number of turns)
    for (size_t first = (size_t)blockIdx.x * GROUPS + (TPR < 32 ? group & ~(32U / TPR - 1U) : group); first < rows; first += stride) {
        const size_t row = TPR < 32 ? first + (group & (32U / (TPR < 32 ? TPR : 32) - 1U)) : first;
        const bool live = row < rows;
        const size_t at = (live ? row : 0) * cols;
        const bool lives[1] = {live};
        const float2 st[1] = {live ? stats[row] : make_float2(0.0f, 0.0f)};
        ln_backward_rows<T, VE, TPR, LN_EPT, 1>(x + at, g + at, dx + at, dx == nullptr ? nullptr : dx + at, 0, lives, add_to_dx, st, wf, sums2, inv_cols, t, cols, sh, flip);
    }
    if (partial == nullptr) return;
    // the groups' sums, added in order
    sums2.template store<VE, TPR>(sums + (size_t)group * 2U * cols, t, cols);
    __syncthreads();
    for (unsigned c = threadIdx.x; c < 2U * cols; c += LN_BWD_THREADS) {
        float v = 0.0f;
#pragma unroll 8
        for (unsigned k = 0; k < GROUPS; ++k) v += sums[(size_t)k * 2U * cols + c];
        partial[(size_t)blockIdx.x * 2U * cols + c] = v;
    }
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

// dw[c] and db[c]: the blocks' partial sums in a fixed order (32 threads a column, every 32nd block each: one load's latency), rounded once.
template <typename T>
__global__ void __launch_bounds__(1024)
layer_norm_merge_kernel(const float *__restrict__ partial, T *__restrict__ dw, T *__restrict__ db, unsigned blocks, size_t cols)
{
    gdb_pdl_sync();
    __shared__ float sh[32][33];
    const unsigned lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const size_t c = (size_t)blockIdx.x * 32U + lane;
    float s = 0.0f;
    if (c < 2U * cols) {
#pragma unroll 8
        for (unsigned k = part; k < blocks; k += 32U) s += __ldcg(&partial[(size_t)k * 2U * cols + c]);
    }
    sh[part][lane] = s;
    __syncthreads();
    if (part == 0 && c < 2U * cols) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += sh[k][lane];
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

// threads of a row: enough for EPT elements each
#define LN_BY_WIDTH(GO, VE, EPT)                                                                                                                                   \
    (a.cols <= 8U * EPT      ? GO(8, VE)                                                                                                                   \
     : a.cols <= 16U * EPT   ? GO(16, VE)                                                                                                                  \
     : a.cols <= 32U * EPT   ? GO(32, VE)                                                                                                                  \
     : a.cols <= 64U * EPT   ? GO(64, VE)                                                                                                                  \
     : a.cols <= 128U * EPT  ? GO(128, VE)                                                                                                                 \
     : a.cols <= 256U * EPT  ? GO(256, VE)                                                                                                                 \
                                : GO(512, VE))

// Tiles of the streaming kernel: rows for all groups of a block, more where rows are short (16 KB a tile keep the copies large) or where
// the tile would not begin on 16 bytes; false where three stages of them do not fit, the pointers are not aligned, or there are too few
// tiles for the ring to be of use (below two a block the direct kernels have the shorter way).
template <typename T, int TPR, int EPT>
bool ln_tiles(const gd_backend *be, const ln_call &a, int streams, ln_stream *st, unsigned *blocks)
{
    if (a.cols > (size_t)TPR * EPT) return false;
    constexpr unsigned GROUPS = LN_THREADS / TPR;
    if (((uintptr_t)a.x | (uintptr_t)a.g | (uintptr_t)a.dx) % 16U != 0U) return false;
    size_t r = GROUPS;
    // backward takes two rows of a group at a time; with the old gradient as a third stream the tiles stay the same, and with them the
    // order of the weight's and the bias's sums
    const int counted = streams > 1 ? 2 : 1;
    if (counted == 2 && 12U * GROUPS * a.cols * sizeof(T) <= LN_RING_BYTES) r *= 2U;
    while (r * a.cols * sizeof(T) % 16U != 0U || (r < 8U * GROUPS && 2U * r * a.cols * sizeof(T) <= 16384U)) r *= 2U;
    const size_t bytes = r * a.cols * sizeof(T), slot = (bytes + 127U) & ~(size_t)127U;
    const size_t stages = LN_RING_BYTES / (slot * streams), tiles = (a.rows + r - 1U) / r;
    if (LN_RING_BYTES / (slot * counted) < 3U || tiles < 2U * (size_t)gdb_usable_sms(be)) return false;
    st->tile_rows = (unsigned)r;
    st->tile_bytes = (unsigned)bytes;
    st->stages = (unsigned)(stages < LN_MAX_STAGES ? stages : LN_MAX_STAGES);
    *blocks = gdb_usable_sms(be);   // (fewer than tiles)
    return true;
}
template <typename T, int TPR, int VE, int EPT, int BWD>
gd_status stream_go(gd_backend *be, const ln_stream &st, unsigned blocks)
{
    auto kern = layer_norm_stream_kernel<T, TPR, VE, EPT, BWD>;
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)LN_RING_BYTES);
        if (e != cudaSuccess) return gdb_fail(be, e, "layer_norm smem attribute");
        ready = true;
    }
    gdb_launch(kern, blocks, LN_THREADS, LN_RING_BYTES, be->stream, st, be->err_flag);
    return gdb_launched(be, BWD ? "layer_norm_backward" : "layer_norm_forward");
}
ln_stream ln_stream_of(const ln_call &a, bool backward, float *partial)
{
    ln_stream st = {};
    st.x = a.x;
    st.g = a.g;
    st.w = a.w;
    st.b = a.b;
    st.out = backward ? a.dx : a.out;
    st.stats = a.stats;
    st.partial = partial;
    st.rows = a.rows;
    st.cols = (unsigned)a.cols;
    st.eps = a.eps;
    return st;
}

// The streaming kernel where it takes the call; GD_ERR_UNSUPPORTED where it does not. Backward, FP32 rows have 8 elements a thread (two
// rows of a group then fit the ring).
template <typename T, int VE, int BWD>
gd_status stream_typed(gd_backend *be, const ln_call &a, float *partial, unsigned *blocks)
{
    constexpr int EPT = sizeof(T) == 2 || BWD == 0 ? 16 : 8;
    ln_stream st = ln_stream_of(a, BWD != 0, partial);
    if (a.cols > 512U * EPT) return GD_ERR_UNSUPPORTED;
#define GO(TPR, V) (ln_tiles<T, TPR, EPT>(be, a, BWD + 1, &st, blocks) ? stream_go<T, TPR, V, EPT, BWD>(be, st, *blocks) : GD_ERR_UNSUPPORTED)
    return LN_BY_WIDTH(GO, VE, EPT);
#undef GO
}

template <typename T, int TPR, int VE>
gd_status fwd_go(gd_backend *be, const ln_call &a)
{
    constexpr unsigned THREADS = ln_fwd_threads(TPR), PER = THREADS / TPR;
    constexpr size_t smem = ln_fwd_smem<T, VE>(TPR);
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(layer_norm_fwd_kernel<T, TPR, VE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return gdb_fail(be, e, "layer_norm_forward smem attribute");
        ready = true;
    }
    // (one wave: blocks stay and walk over the rows)
    const size_t most = (size_t)gdb_usable_sms(be) * ln_fwd_blocks(TPR, VE), need = (a.rows + PER - 1U) / PER;
    gdb_launch(layer_norm_fwd_kernel<T, TPR, VE>, (unsigned)(need < most ? need : most), THREADS, smem, be->stream, (const T *)a.x, (const T *)a.w, (const T *)a.b, (T *)a.out,
               a.stats, a.rows, (unsigned)a.cols, a.eps);
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
    if (!vec) {
        unsigned blocks;
        const gd_status st = stream_typed<T, 1, 0>(be, a, nullptr, &blocks);
        if (st != GD_ERR_UNSUPPORTED) return st;
    }
#define GO(TPR, V) fwd_go<T, TPR, V>(be, a)
    return vec ? LN_BY_WIDTH(GO, VE, LN_EPT) : LN_BY_WIDTH(GO, 1, LN_EPT);
#undef GO
}

template <typename T, int TPR, int VE>
gd_status bwd_go(gd_backend *be, const ln_call &a, float *partial, unsigned max_blocks, unsigned *blocks)
{
    constexpr unsigned PER = LN_BWD_THREADS / TPR;
    const size_t need = (a.rows + PER - 1U) / PER;
    *blocks = (unsigned)(need < max_blocks ? need : max_blocks);
    const int smem = (int)(PER * 2U * a.cols * sizeof(float));   // (64 KB at most)
    static bool ready = false;
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(layer_norm_bwd_kernel<T, TPR, VE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(PER * 2U * TPR * LN_EPT * sizeof(float)));
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
        if (sums) {   // (first: dx may take g's place)
            const size_t col_blocks = (a.cols + 255U) / 256U;
            size_t chunks = ((size_t)be->sm_count * 8U + col_blocks - 1U) / col_blocks;
            if (chunks > fit) chunks = fit;
            if (chunks > a.rows) chunks = a.rows;
            if (chunks > 65535U) chunks = 65535U;
            if (col_blocks > 0x7fffffffU) return GD_ERR_UNSUPPORTED;
            const size_t per = (a.rows + chunks - 1U) / chunks;
            blocks = (unsigned)((a.rows + per - 1U) / per);
            gdb_launch(layer_norm_columns_long_kernel<T>, dim3((unsigned)col_blocks, blocks), 256, 0, be->stream, (const T *)a.x, (const float2 *)a.stats, (const T *)a.g, partial,
                       a.rows, a.cols, per);
            st = gdb_launched(be, "layer_norm_backward columns");
            if (st != GD_OK) return st;
        }
        if (a.dx != nullptr) {
            gdb_launch(layer_norm_bwd_long_kernel<T>, gdb_grid_for(a.rows, 1U, be, 4U), 512, 0, be->stream, (const T *)a.x, (const T *)a.w, (const float2 *)a.stats, (const T *)a.g,
                       (T *)a.dx, a.add_to_dx, a.rows, a.cols);
            st = gdb_launched(be, "layer_norm_backward");
            if (st != GD_OK) return st;
        }
        st = GD_OK;
    } else {
        const unsigned sms = gdb_usable_sms(be), most = !sums || fit > sms ? sms : (unsigned)fit;
        const bool vec = a.cols % VE == 0U && (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.g | (uintptr_t)a.dx) % 16U) == 0U;
        st = most < sms                    ? GD_ERR_UNSUPPORTED
             : a.add_to_dx                 ? (vec ? stream_typed<T, VE, 2>(be, a, partial, &blocks) : stream_typed<T, 1, 2>(be, a, partial, &blocks))
                                           : (vec ? stream_typed<T, VE, 1>(be, a, partial, &blocks) : stream_typed<T, 1, 1>(be, a, partial, &blocks));
        if (st == GD_ERR_UNSUPPORTED) {
#define GO(TPR, V) bwd_go<T, TPR, V>(be, a, partial, most, &blocks)
            st = vec ? LN_BY_WIDTH(GO, VE, LN_EPT) : LN_BY_WIDTH(GO, 1, LN_EPT);
#undef GO
        }
    }
    if (st != GD_OK || !sums) return st;
    gdb_launch(layer_norm_merge_kernel<T>, (unsigned)((2U * a.cols + 31U) / 32U), 1024, 0, be->stream, (const float *)partial, (T *)a.dw, (T *)a.db, blocks, a.cols);
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
        !ln_ptr(grad_bias, x->dtype, args->cols, &dbp) || ((uintptr_t)sp % 8U) != 0U || (accumulate != 0 && dxp == gp)) {
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
    a.add_to_dx = accumulate != 0 && dxp != NULL;
    return x->dtype == GDB_DTYPE_F16 ? bwd_typed<__half>(be, a) : (x->dtype == GDB_DTYPE_BF16 ? bwd_typed<__nv_bfloat16>(be, a) : bwd_typed<float>(be, a));
}

}  // extern "C"
