// The elementwise halves of a Muon step, around gdb200_orthogonalize: the momentum before it, the update of the weights behind it.
//
//   g = grad * grad_scale,  m <- mu m + g,  d = g + mu m (Nesterov) or m          muon_momentum_kernel
//   o = orthogonalize(d)
//   p <- p - step o - decay p,  param = round(p)                                  muon_apply_kernel
//
// Both are bound by HBM: with 16-bit gradients and parameters 14 and 12 bytes an element (momentum, direction and master FP32, the update
// 16 bits), a flop or two for each: 4 matrices of 2048 x 5632 take 103 us (6.2 TB/s) and 89 us (6.2 TB/s), 12 of 512 x 512 (in L2) 11 and 8 us,
// of steps of 1.7 and 0.22 ms. One launch takes up to MUON_BATCH tensors, so that the matrices of a model need a few launches a step;
// a block has 2048 consecutive elements of one tensor, 8 a thread in 16-byte accesses. The direction is FP32: an unscaled gradient may lie
// below FP16's range, and what is orthogonalised is scaled by its own norm only afterwards.
#include "common.cuh"

#include <string.h>

namespace {

constexpr int MUON_BATCH = 48;             // (the items below stay under the 4 KB of kernel parameters that a launch takes by the short path)
constexpr unsigned MUON_ELEMS = 2048U;     // elements of a block

struct muon_momentum_item {
    const void *grad;
    float *momentum, *direction;
    const float *grad_scale;   // nullable
    const int *found_inf;      // nullable
    size_t count;
    uint32_t grad_dtype;
    int nesterov;
    float mu;
};
struct muon_apply_item {
    void *param;
    float *master;             // nullable
    const void *update;
    const int *found_inf;      // nullable
    unsigned *param_step, *optimizer_step;   // nullable
    size_t count;
    uint32_t param_dtype, update_dtype;
    float step, decay;
};
template <typename ITEM>
struct muon_batch {
    ITEM it[MUON_BATCH];
    unsigned block_start[MUON_BATCH + 1];
    int n;
};
static_assert(sizeof(muon_batch<muon_momentum_item>) <= 4000 && sizeof(muon_batch<muon_apply_item>) <= 4000, "kernel parameters");

// 8 values of any floating dtype from and to a 16-byte boundary
__device__ __forceinline__ void load8(const void *p, size_t i, uint32_t dtype, float (&v)[8])
{
    if (dtype == GDB_DTYPE_F32) {
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>((const float *)p + i);
        *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>((const float *)p + i + 4);
        return;
    }
    const uint4 raw = *reinterpret_cast<const uint4 *>((const unsigned short *)p + i);
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned short bits = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
        v[e] = dtype == GDB_DTYPE_F16 ? gdb_io<__half>::up(bits) : gdb_io<__nv_bfloat16>::up(bits);
    }
}
__device__ __forceinline__ void store8(void *p, size_t i, uint32_t dtype, const float (&v)[8])
{
    if (dtype == GDB_DTYPE_F32) {
        *reinterpret_cast<float4 *>((float *)p + i) = *reinterpret_cast<const float4 *>(v);
        *reinterpret_cast<float4 *>((float *)p + i + 4) = *reinterpret_cast<const float4 *>(v + 4);
        return;
    }
    unsigned w[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const unsigned lo = dtype == GDB_DTYPE_F16 ? gdb_io<__half>::down(v[e]) : gdb_io<__nv_bfloat16>::down(v[e]);
        const unsigned hi = dtype == GDB_DTYPE_F16 ? gdb_io<__half>::down(v[e + 1]) : gdb_io<__nv_bfloat16>::down(v[e + 1]);
        w[e >> 1] = (lo & 0xffffU) | hi << 16;
    }
    *reinterpret_cast<uint4 *>((unsigned short *)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float load1(const void *p, size_t i, uint32_t dtype)
{
    return dtype == GDB_DTYPE_F16 ? __half2float(((const __half *)p)[i]) : (dtype == GDB_DTYPE_BF16 ? __bfloat162float(((const __nv_bfloat16 *)p)[i]) : ((const float *)p)[i]);
}
__device__ __forceinline__ void store1(void *p, size_t i, uint32_t dtype, float v)
{
    if (dtype == GDB_DTYPE_F16) ((__half *)p)[i] = __float2half_rn(v);
    else if (dtype == GDB_DTYPE_BF16) ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
    else ((float *)p)[i] = v;
}

template <typename ITEM>
__device__ __forceinline__ int muon_item_of_block(const muon_batch<ITEM> &b)
{
    int t = 0;
    while (t + 1 < b.n && blockIdx.x >= b.block_start[t + 1]) ++t;
    return t;
}

__global__ void __launch_bounds__(256) muon_momentum_kernel(const __grid_constant__ muon_batch<muon_momentum_item> b)
{
    gdb_pdl_sync();
    const int t = muon_item_of_block(b);
    const muon_momentum_item &a = b.it[t];
    // an overflow somewhere: the momentum stays, the direction is one that the next kernel can read
    const bool skip = a.found_inf != nullptr && *a.found_inf != 0;
    const float gs = a.grad_scale != nullptr ? a.grad_scale[0] : 1.0f;
    const size_t base = (size_t)(blockIdx.x - b.block_start[t]) * MUON_ELEMS;
    auto element = [&](float g, float &m) {
        g = gs == 0.0f ? 0.0f : __fmul_rn(g, gs);
        m = fmaf(a.mu, m, g);
        return a.nesterov ? fmaf(a.mu, m, g) : m;
    };
    if (base + MUON_ELEMS <= a.count && (((uintptr_t)a.grad | (uintptr_t)(a.momentum) | (uintptr_t)(a.direction)) % 16U) == 0U) {
        const size_t i = base + (size_t)threadIdx.x * 8U;
        float g[8], m[8], d[8];
        if (skip) {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = 0.0f;
        } else {
            load8(a.grad, i, a.grad_dtype, g);
            load8(a.momentum, i, GDB_DTYPE_F32, m);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = element(g[e], m[e]);
            store8(a.momentum, i, GDB_DTYPE_F32, m);
        }
        store8(a.direction, i, GDB_DTYPE_F32, d);
        return;
    }
    const size_t end = base + MUON_ELEMS < a.count ? base + MUON_ELEMS : a.count;
    for (size_t i = base + threadIdx.x; i < end; i += 256U) {
        float m = a.momentum[i];
        const float d = element(load1(a.grad, i, a.grad_dtype), m);
        if (!skip) a.momentum[i] = m;
        a.direction[i] = skip ? 0.0f : d;
    }
}

__global__ void __launch_bounds__(256) muon_apply_kernel(const __grid_constant__ muon_batch<muon_apply_item> b)
{
    gdb_pdl_sync();
    const int t = muon_item_of_block(b);
    const muon_apply_item &a = b.it[t];
    if (a.found_inf != nullptr && *a.found_inf != 0) return;
    if (blockIdx.x == b.block_start[t] && threadIdx.x == 0) {   // (read by nobody in this launch)
        if (a.param_step != nullptr) a.param_step[0] += 1U;
        if (a.optimizer_step != nullptr) a.optimizer_step[0] += 1U;
    }
    const size_t base = (size_t)(blockIdx.x - b.block_start[t]) * MUON_ELEMS;
    auto element = [&](float p, float o) { return __fsub_rn(__fsub_rn(p, __fmul_rn(a.step, o)), __fmul_rn(a.decay, p)); };
    void *state = a.master != nullptr ? (void *)a.master : a.param;
    const uint32_t state_dtype = a.master != nullptr ? (uint32_t)GDB_DTYPE_F32 : a.param_dtype;
    if (base + MUON_ELEMS <= a.count && (((uintptr_t)a.param | (uintptr_t)a.master | (uintptr_t)a.update) % 16U) == 0U) {
        const size_t i = base + (size_t)threadIdx.x * 8U;
        float p[8], o[8];
        load8(state, i, state_dtype, p);
        load8(a.update, i, a.update_dtype, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = element(p[e], o[e]);
        if (a.master != nullptr) store8(a.master, i, GDB_DTYPE_F32, p);
        store8(a.param, i, a.param_dtype, p);
        return;
    }
    const size_t end = base + MUON_ELEMS < a.count ? base + MUON_ELEMS : a.count;
    for (size_t i = base + threadIdx.x; i < end; i += 256U) {
        const float p = element(load1(state, i, state_dtype), load1(a.update, i, a.update_dtype));
        if (a.master != nullptr) a.master[i] = p;
        store1(a.param, i, a.param_dtype, p);
    }
}

// count elements of `bytes` each at `offset` of the buffer, aligned to an element
bool part(gd_backend_buffer *buffer, size_t offset, uint64_t count, size_t bytes, unsigned char **p)
{
    if (!gdb_range_ok(buffer, offset, count * bytes)) return false;
    *p = buffer->dptr + offset;
    return ((uintptr_t)*p % bytes) == 0U;
}
bool part_or_null(gd_backend_buffer *buffer, size_t offset, uint64_t count, size_t bytes, unsigned char **p)
{
    *p = NULL;
    return buffer == NULL || part(buffer, offset, count, bytes, p);
}

gd_status fill(const gdb200_muon_desc *d, muon_momentum_item *it)
{
    unsigned char *grad, *momentum, *direction, *scale, *found;
    if (!gdb_is_float_dtype(d->grad_dtype)) return GD_ERR_UNSUPPORTED;
    if (d->count == 0U || d->count > (1ULL << 40) || !part(d->grad_buffer, d->grad_offset, d->count, gdb_dtype_size(d->grad_dtype), &grad) ||
        !part(d->momentum_buffer, d->momentum_offset, d->count, 4U, &momentum) || !part(d->direction_buffer, d->direction_offset, d->count, 4U, &direction) ||
        !part_or_null(d->grad_scale_buffer, d->grad_scale_offset, 1U, 4U, &scale) || !part_or_null(d->found_inf_buffer, d->found_inf_offset, 1U, 4U, &found)) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    *it = {grad, (float *)momentum, (float *)direction, (const float *)scale, (const int *)found, (size_t)d->count, d->grad_dtype, d->nesterov != 0, d->momentum};
    return GD_OK;
}
gd_status fill(const gdb200_muon_desc *d, muon_apply_item *it)
{
    unsigned char *param, *master, *update, *found, *param_step = NULL, *optimizer_step = NULL;
    if (!gdb_is_float_dtype(d->param_dtype) || !gdb_is_float_dtype(d->update_dtype)) return GD_ERR_UNSUPPORTED;
    if (d->count == 0U || d->count > (1ULL << 40) || !part(d->param_buffer, d->param_offset, d->count, gdb_dtype_size(d->param_dtype), &param) ||
        !part_or_null(d->master_buffer, d->master_offset, d->count, 4U, &master) ||
        !part(d->update_buffer, d->update_offset, d->count, gdb_dtype_size(d->update_dtype), &update) ||
        !part_or_null(d->found_inf_buffer, d->found_inf_offset, 1U, 4U, &found) || !part_or_null(d->steps_buffer, d->param_step_offset, 1U, 4U, &param_step) ||
        (d->update_optimizer_step && (d->steps_buffer == NULL || !part(d->steps_buffer, d->optimizer_step_offset, 1U, 4U, &optimizer_step)))) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    *it = {param, (float *)master, update, (const int *)found, (unsigned *)param_step, (unsigned *)optimizer_step, (size_t)d->count, d->param_dtype, d->update_dtype, d->step, d->decay};
    return GD_OK;
}

template <typename ITEM>
gd_status run(gd_backend *be, const gdb200_muon_desc *descs, uint32_t n, void (*kernel)(const muon_batch<ITEM>), const char *what)
{
    if (be == NULL || (n != 0U && descs == NULL)) return GD_ERR_INVALID_ARGUMENT;
    for (uint32_t i = 0; i < n; ++i) {   // all of them before the first launch: a bad one leaves nothing half done
        ITEM it;
        const gd_status st = fill(&descs[i], &it);
        if (st != GD_OK) return st;
    }
    for (uint32_t start = 0; start < n;) {
        muon_batch<ITEM> b;
        memset(&b, 0, sizeof(b));
        uint64_t blocks = 0;
        while (start < n && b.n < MUON_BATCH) {
            const uint64_t more = (descs[start].count + MUON_ELEMS - 1U) / MUON_ELEMS;
            if (blocks + more > 0x7fffffffU) break;   // (one tensor has 2^29 blocks at most)
            (void)fill(&descs[start++], &b.it[b.n]);
            b.block_start[b.n++] = (unsigned)blocks;
            blocks += more;
        }
        b.block_start[b.n] = (unsigned)blocks;
        gdb_launch(kernel, (unsigned)blocks, 256, 0, be->stream, b);
        const gd_status st = gdb_launched(be, what);
        if (st != GD_OK) return st;
    }
    return GD_OK;
}

}  // namespace

extern "C" {

gd_status gdb200_muon_momentum_batch(gd_backend *be, const gdb200_muon_desc *descs, uint32_t desc_count)
{
    return run<muon_momentum_item>(be, descs, desc_count, muon_momentum_kernel, "muon momentum");
}

gd_status gdb200_muon_apply_batch(gd_backend *be, const gdb200_muon_desc *descs, uint32_t desc_count)
{
    return run<muon_apply_item>(be, descs, desc_count, muon_apply_kernel, "muon apply");
}

}  // extern "C"
