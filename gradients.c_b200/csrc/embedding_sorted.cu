// Embedding lookup with a scale, and its gradient summed in token order.
//
//   out[i] = s table[ids[i]];   d_table[v] = s * (sum over i with ids[i] = v, i ascending, of g[i])
//
// HBM-bound: the gradient reads g once and writes every table row once. The scatter with FP32 atomics next door (embedding_rope.cu)
// needs a table of vocab x dim floats that is cleared before and rounded after, and its sums change from run to run; here the
// positions are sorted by token first and a row is written once, when its sum is complete.
//
// 1. es_sort_kernel: a stable counting sort of the positions in one launch without communication between blocks. A block owns a slice
//    of the vocabulary and reads ALL ids (they lie in L2: 4 bytes each against 2 dim for the gradient's row), so it knows by itself how
//    many ids lie below its slice. It also clears the rows of its slice that no id names.
// 2. es_reduce_kernel: equal pieces of the sorted list, whatever the frequencies: a warp adds a few rows up to a few dozen for 32 vectors of
//    columns, runs that begin and end within a piece are written, the others go to FP32 partial sums, which the block of the piece where
//    the run ends adds up in order.
// Every sum is FP32 in an order that depends on the ids, the sizes, the number of SMs and the workspace alone.
// 16384 ids, 32768 x 2048 BF16: lookup 19.5 us (6.2 TB/s), 1. 24 (14 of them clear 80 MB), 2. 25.5 (4.7 TB/s); 18432 ids, 2048 x 512 FP16: 6, 9.5,
// 13, where launches and the waits between pieces count. The scatter next door and this on the same inputs, calls among others: 128 and 46 us,
// 39 and 20, 5003 ids of 20011 x 321 FP32 37 and 21.
#include "common.cuh"

#include <type_traits>

namespace {

constexpr int ES_SORT_WARPS = 32, ES_AHEAD = 8;   // (ids on their way, a lane)
constexpr unsigned ES_MAX_WIDTH = 1536, ES_ZEROS = 4096, ES_SORT_SMEM = 220 * 1024;   // tokens of a slice (32 x 1536 counters fill 192 KB), bytes
constexpr int ES_WARPS = 8, ES_BLOCKS = 4;   // of a summing block; blocks on an SM
constexpr unsigned ES_POLLS = 1U << 21;      // of a flag, a second or two, before a wait gives up

template <typename T, int VE> struct es_vec {
    T v[VE];
};
template <> struct __align__(16) es_vec<__half, 8> { __half v[8]; };
template <> struct __align__(16) es_vec<__nv_bfloat16, 8> { __nv_bfloat16 v[8]; };
template <> struct __align__(16) es_vec<float, 4> { float v[4]; };

// ------------------------------------------------------------------ forward
// round(scale * v) of the elements of 16 bytes, two 16-bit ones at a time, or of one element
template <typename T>
__device__ __forceinline__ uint4 es_scaled(uint4 v, float scale)
{
    unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4U) {
            w[k] = __float_as_uint(__uint_as_float(w[k]) * scale);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
            *reinterpret_cast<__half2 *>(&w[k]) = __floats2half2_rn(f.x * scale, f.y * scale);
        } else {
            *reinterpret_cast<__nv_bfloat162 *>(&w[k]) = __floats2bfloat162_rn(__uint_as_float(w[k] << 16) * scale, __uint_as_float(w[k] & 0xffff0000U) * scale);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ T es_scaled(T v, float scale)
{
    T r;
    gdb_io<T>::st(&r, 0, gdb_io<T>::ld(&v, 0) * scale);
    return r;
}

// LANES threads per row, ROWS rows each in flight; V: uint4 where rows are whole 16-byte vectors, else T.
template <typename T, typename V, int LANES>
__global__ void __launch_bounds__(256)
es_lookup_kernel(const V *__restrict__ table, const int *__restrict__ ids, V *__restrict__ out, size_t n, size_t vocab, size_t vecs, float scale)
{
    gdb_pdl_sync();
    constexpr int ROWS = 4, PER = 256 / LANES;
    const unsigned t = threadIdx.x % LANES, r = threadIdx.x / LANES;
    for (size_t first = (size_t)blockIdx.x * PER * ROWS; first < n; first += (size_t)gridDim.x * PER * ROWS) {
        int id[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const size_t row = first + u * PER + r;
            id[u] = row < n ? __ldg(&ids[row]) : -1;
        }
        for (size_t v = t; v < vecs; v += LANES) {
            V a[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                if (id[u] >= 0 && (size_t)id[u] < vocab) a[u] = __ldg(table + (size_t)id[u] * vecs + v); else a[u] = V{};
            }
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                const size_t row = first + u * PER + r;
                const bool in = id[u] >= 0 && (size_t)id[u] < vocab;
                if (row < n) out[row * vecs + v] = es_scaled<T>(a[u], in ? scale : __int_as_float(0x7fc00000));   // (a row of NaN)
            }
        }
    }
}

// ------------------------------------------------------------------ sort
// Block b owns tokens [b * width, (b + 1) * width). order[k] = position of the k-th id in token order, token[k] = that id; count[0] = ids
// inside the table. `clear` != NULL: the gradient table, whose rows without an id are set to zero. A warp notes up to `notes` ids of the
// slice, so that only a warp with more (of a frequent token) has to look at its ids again: what bounds the kernel is the instructions
// that every block spends on every id. Whole vectors are cleared by bulk copies of zeros beside the sorting.
template <typename V>
__global__ void __launch_bounds__(ES_SORT_WARPS * 32)
es_sort_kernel(const int *__restrict__ ids, unsigned n, unsigned vocab, unsigned width, unsigned notes, unsigned *__restrict__ order, int *__restrict__ token,
               unsigned *__restrict__ count, unsigned *__restrict__ flags, unsigned n_flags, V *__restrict__ clear, size_t row_vecs)
{
    gdb_pdl_sync();
    constexpr bool BULK = sizeof(V) == 16U;
    extern __shared__ uint2 sort_smem[];     // notes: [warps, notes] (position, token - v0); counters [warps, width], then places
    __shared__ unsigned warp_sum[ES_SORT_WARPS], below_sum[ES_SORT_WARPS], absent[ES_MAX_WIDTH / 32U];   // absent: a bit per token without an id
    __shared__ __align__(128) uint4 zeros[BULK ? ES_ZEROS / 16U : 1U];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned v0 = blockIdx.x * width, w = min(width, vocab - v0);
    uint2 *note = sort_smem + (size_t)warp * notes;
    unsigned *counters = reinterpret_cast<unsigned *>(sort_smem + (size_t)ES_SORT_WARPS * notes), *mine = counters + (size_t)warp * width;
    for (unsigned k = threadIdx.x; k < ES_SORT_WARPS * width; k += blockDim.x) counters[k] = 0U;
    for (unsigned k = blockIdx.x * blockDim.x + threadIdx.x; k < n_flags; k += gridDim.x * blockDim.x) flags[k] = 0U;
    if constexpr (BULK) {
        if (threadIdx.x < ES_ZEROS / 16U) zeros[threadIdx.x] = make_uint4(0U, 0U, 0U, 0U);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    // a warp reads a range of the ids, 32 at a time
    const unsigned per = ((n + ES_SORT_WARPS * 32U - 1U) / (ES_SORT_WARPS * 32U)) * 32U;
    const unsigned i0 = min(n, warp * per), i1 = min(n, i0 + per);
    unsigned below = 0U, found = 0U;
    const unsigned lower = (1U << lane) - 1U;
    for (unsigned i = i0; i < i1; i += 32U * ES_AHEAD) {
        unsigned id[ES_AHEAD];
#pragma unroll
        for (int u = 0; u < ES_AHEAD; ++u) id[u] = i + 32U * u + lane < i1 ? (unsigned)__ldg(&ids[i + 32U * u + lane]) : 0xffffffffU;
#pragma unroll
        for (int u = 0; u < ES_AHEAD; ++u) {
            below += id[u] < v0 ? 1U : 0U;   // (a negative id lies above every vocabulary)
            const unsigned k = id[u] - v0, here = __ballot_sync(0xffffffffU, k < w);
            if (here == 0U) continue;
            if (k < w) {
                atomicAdd(&mine[k], 1U);
                const unsigned at = found + __popc(here & lower);
                if (at < notes) note[at] = make_uint2(i + 32U * u + lane, k);
            }
            found += __popc(here);
        }
    }
    below = __reduce_add_sync(0xffffffffU, below);
    if (lane == 0) below_sum[warp] = below;
    __syncthreads();
    unsigned base = __reduce_add_sync(0xffffffffU, below_sum[lane]);
    // place of the first id of (token, warp), tokens first: a thread per token, 1024 tokens at a time
    for (unsigned k0 = 0; k0 < w; k0 += blockDim.x) {
        const unsigned k = k0 + threadIdx.x;
        unsigned total = 0U;
        if (k < w) {
#pragma unroll 8
            for (int s = 0; s < ES_SORT_WARPS; ++s) total += counters[(size_t)s * width + k];
        }
        unsigned incl = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned up = __shfl_up_sync(0xffffffffU, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        const unsigned sums = warp_sum[lane], all = __reduce_add_sync(0xffffffffU, sums);
        const unsigned before = base + __reduce_add_sync(0xffffffffU, lane < warp ? sums : 0U);
        if (k < w) {
            unsigned at = before + incl - total;
#pragma unroll 8
            for (int s = 0; s < ES_SORT_WARPS; ++s) {
                const unsigned c = counters[(size_t)s * width + k];
                counters[(size_t)s * width + k] = at;
                at += c;
            }
            if constexpr (BULK) {
                if (clear != nullptr && total == 0U) {
                    V *row = clear + (size_t)(v0 + k) * row_vecs;
                    const unsigned from = (unsigned)__cvta_generic_to_shared(zeros);
                    for (size_t c = 0; c < row_vecs; c += ES_ZEROS / 16U) {
                        const unsigned bytes = (unsigned)min(row_vecs - c, (size_t)(ES_ZEROS / 16U)) * 16U;
                        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(row + c), "r"(from), "r"(bytes) : "memory");
                    }
                }
            }
        }
        const unsigned none = __ballot_sync(0xffffffffU, k < w && total == 0U);
        if (!BULK && lane == 0 && k0 + warp * 32U < w) absent[k0 / 32U + warp] = none;
        base += all;
        __syncthreads();
    }
    if constexpr (BULK) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    if (blockIdx.x == gridDim.x - 1U && threadIdx.x == 0) {
        count[0] = base;
        count[1] = 0U;   // the summing blocks' turns
    }
    // every id of the slice to its place, equal ids of a warp's 32 in lane order
    const auto put = [&](bool in, unsigned pos, unsigned k) {
        // lanes with the same token, a bit of it at a time (a match instruction took three times as long)
        unsigned peers = __ballot_sync(0xffffffffU, in);
        for (unsigned bit = 1U; bit < w; bit <<= 1) {
            const unsigned set = __ballot_sync(0xffffffffU, (k & bit) != 0U);
            peers &= (k & bit) != 0U ? set : ~set;
        }
        const unsigned before = __popc(peers & lower);
        unsigned at = 0U;
        if (in) at = mine[k] + before;
        __syncwarp();
        if (in && before == 0U) mine[k] = at + __popc(peers);
        __syncwarp();
        if (in) {
            order[at] = pos;
            token[at] = (int)(v0 + k);
        }
    };
    const auto put_notes = [&](unsigned held) {
        __syncwarp();
        for (unsigned j = 0; j < held; j += 32U) {
            const bool in = j + lane < held;
            const uint2 e = in ? note[j + lane] : make_uint2(0U, 0U);
            put(in, e.x, e.y);
        }
        __syncwarp();
    };
    if (found <= notes) {
        put_notes(found);
    } else {
        // noted again, and put down whenever the notes are full (the few of every 32 ids by themselves: 300000 ids, 32000 tokens, 232 instead of 138 us)
        unsigned held = 0U;
        for (unsigned i = i0; i < i1; i += 32U * ES_AHEAD) {
            unsigned id[ES_AHEAD];
#pragma unroll
            for (int u = 0; u < ES_AHEAD; ++u) id[u] = i + 32U * u + lane < i1 ? (unsigned)__ldg(&ids[i + 32U * u + lane]) : 0xffffffffU;
#pragma unroll 1
            for (int u = 0; u < ES_AHEAD; ++u) {
                const unsigned k = id[0] - v0, here = __ballot_sync(0xffffffffU, k < w);   // (the array moves on: its places are registers)
#pragma unroll
                for (int m = 1; m < ES_AHEAD; ++m) id[m - 1] = id[m];
                if (k < w) note[held + __popc(here & lower)] = make_uint2(i + 32U * u + lane, k);
                held += __popc(here);
                if (held + 32U > notes) {
                    put_notes(held);
                    held = 0U;
                }
            }
        }
        put_notes(held);
    }
    if constexpr (BULK) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else if (clear != nullptr) {
        // neighbouring rows together, whole vectors in the middle; 32 tokens a warp, or several warps where there are fewer
        const unsigned words = (w + 31U) / 32U, share = words < ES_SORT_WARPS ? ES_SORT_WARPS / words : 1U;
        for (unsigned unit = warp; unit < words * share; unit += ES_SORT_WARPS) {
            const unsigned k0 = unit % words * 32U, part = unit / words;
            unsigned bits = absent[k0 / 32U];
            while (bits != 0U) {
                const unsigned r = __ffs((int)bits) - 1U, stop = ~(bits >> r), rows = stop != 0U ? __ffs((int)stop) - 1U : 32U;
                bits &= r + rows < 32U ? 0xffffffffU << (r + rows) : 0U;
                V *p = clear + (size_t)(v0 + k0 + r) * row_vecs;
                const size_t n_all = (size_t)rows * row_vecs, lead = (16U - (uintptr_t)p % 16U) % 16U / sizeof(V), n_lead = lead < n_all ? lead : n_all;
                const size_t n_wide = (n_all - n_lead) / (16U / sizeof(V)), behind = n_lead + n_wide * (16U / sizeof(V));
                const V zero = {};
                for (size_t c = part * 32U + lane; c < n_wide; c += share * 32U) reinterpret_cast<uint4 *>(p + n_lead)[c] = make_uint4(0U, 0U, 0U, 0U);
                if (part == 0U && lane < n_lead) p[lane] = zero;
                if (part == 0U && behind + lane < n_all) p[behind + lane] = zero;
            }
        }
    }
}

// ------------------------------------------------------------------ sums
template <typename T, int VE>
__device__ __forceinline__ void es_store(T *p, const float *s, float scale, bool add)
{
    typedef es_vec<T, VE> vec;
    vec v;
    if (add) v = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        // accumulating: round, add, round, as gd_backend_accumulate after the plain call would
        const float r = __fmul_rn(s[e], scale);   // (never fused with the addition)
        gdb_io<T>::st(v.v, e, add ? gdb_io<T>::ld(v.v, e) + gdb_io<T>::rnd(r) : r);
    }
    *reinterpret_cast<vec *>(p) = v;
}

__device__ __forceinline__ unsigned es_load_acquire(const unsigned *p)
{
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// Piece c, slab s: sorted entries [c * piece, (c + 1) * piece), a warp an eighth of them, columns [s * 32 * VE * NV, ...). The piece in which
// a run ends adds up its parts: partial[b, 1] of the piece b where it begins, partial[k, 0] of those that it fills, its own. Blocks take
// their pieces in the order in which they start, so a block waits only for ones that run already (a launch of its own for the parts, 18432 ids
// of 2048 x 512 FP16 26.9 instead of 27.4 us, 5003 of 20011 x 321 FP32 27.4 instead of 25.5, 16384 of 32768 x 2048 BF16 69.0 instead of 66.5);
// flags[c, s]: the parts of piece c are in memory.
template <typename T, int VE, int NV>
__global__ void __launch_bounds__(ES_WARPS * 32, ES_BLOCKS)
es_reduce_kernel(const T *__restrict__ g, const unsigned *__restrict__ order, const int *__restrict__ token, unsigned *count, T *__restrict__ table, float *partial,
                 unsigned *flags, unsigned n, unsigned piece, unsigned slabs, size_t dim, float scale, bool add, int *err_flag)
{
    gdb_pdl_sync();
    typedef es_vec<T, VE> vec;
    // Whole vectors travel through shared memory, ES_AHEAD_ROWS rows on their way: a thread copies and reads its own 16 bytes. (As registers
    // the rows of a ring share the few scoreboards of a warp, and waiting for one waits for those asked for last as well: 34 to 54 us
    // where this takes 24, 16384 rows of 2048 BF16.) Single elements are fetched four rows at a time.
    constexpr bool ASYNC = sizeof(vec) == 16U;
    constexpr int COLS = 32 * VE * NV, SLOTS = 8, U = ASYNC ? SLOTS - 1 : 2;
    static_assert(!ASYNC || NV == 1, "one vector per lane and row");
    __shared__ float head[ES_WARPS][COLS];
    __shared__ __align__(16) unsigned char ring[ES_WARPS][ASYNC ? SLOTS * 512 : COLS * 4];   // (its beginning holds the warp's last sums behind the loop)
    const auto tail = [&](int w) { return reinterpret_cast<float *>(ring[w]); };
    // of each warp's entries: the first token, and whether its run began before them (1), goes on behind them (2), does both with one token (4);
    // 8: there are none
    __shared__ int first_token[ES_WARPS];
    __shared__ unsigned ends[ES_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    static_assert(COLS <= ES_WARPS * 32, "a thread per column");
    __shared__ unsigned turn;
    if (threadIdx.x == 0) turn = atomicAdd(&count[1], 1U);
    __syncthreads();
    const unsigned chunk = turn / slabs, slab = turn - chunk * slabs, e0 = chunk * piece, per = piece / ES_WARPS, a = e0 + warp * per;
    // (all n places of the lists may be read; those behind the ids inside the table hold nothing that is used)
    unsigned mine = a + lane < n ? __ldg(&order[a + lane]) : 0U;
    int mine_token = a + lane < n ? __ldg(&token[a + lane]) : -1;
    const int token_before = a > 0U && a <= n ? __ldg(&token[a - 1U]) : -1, token_after = a + per < n ? __ldg(&token[a + per]) : -1;
    const unsigned total = __ldcg(count);
    if (e0 >= total) return;
    const unsigned e1 = min(total, e0 + piece), b = min(e1, a + per);
    const bool some = a < b;
    const size_t col0 = (size_t)slab * COLS;
    float acc[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[j][e] = 0.0f;
    }
    auto keep = [&](float *to) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                to[(lane + 32 * j) * VE + e] = acc[j][e];
                acc[j][e] = 0.0f;
            }
        }
    };
    // runs that are not complete within the warp's entries
    const int begin = __shfl_sync(0xffffffffU, mine_token, 0), after = b < total ? token_after : -1;
    bool open_left = some && token_before == begin;
    int current = begin;
    auto finish = [&] {
        if (open_left) {
            keep(head[warp]);
            open_left = false;
            return;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const size_t c = col0 + (lane + 32 * j) * VE;
            if (c < dim) es_store<T, VE>(table + (size_t)current * dim + c, acc[j], scale, add);
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[j][e] = 0.0f;
        }
    };
    for (unsigned i = a; i < b; i += 32U) {
        if (i != a) {
            mine = i + lane < b ? order[i + lane] : 0U;
            mine_token = i + lane < b ? token[i + lane] : -1;
        }
        const int here = (int)min(32U, b - i);
        const auto add_row = [&](int q, const vec *row) {
            const int tok = __shfl_sync(0xffffffffU, mine_token, q);
            if (tok != current) {
                finish();
                current = tok;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (col0 + (lane + 32 * j) * VE < dim) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[j][e] += gdb_io<T>::ld(row[j].v, e);
                }
            }
        };
        if constexpr (ASYNC) {
            const bool inside = col0 + lane * VE < dim;
            const unsigned slots = (unsigned)__cvta_generic_to_shared(ring[warp]) + 16U * lane;
            const T *column = g + col0 + lane * VE;
            const auto fetch = [&](int q) {
                const unsigned pos = __shfl_sync(0xffffffffU, mine, q & 31);
                if (q < here && inside) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slots + 512U * (q % SLOTS)), "l"(column + (size_t)pos * dim) : "memory");
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll
            for (int q = 0; q < U; ++q) fetch(q);
#pragma unroll 1
            for (int q = 0; q < here; ++q) {
                asm volatile("cp.async.wait_group %0;" ::"n"(U - 1) : "memory");
                const vec row = *reinterpret_cast<const vec *>(ring[warp] + 512 * (q % SLOTS) + 16 * lane);
                add_row(q, &row);
                fetch(q + U);   // (to the place that was read one row ago)
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        } else {
            for (int q = 0; q < here; q += U) {
                vec v[U][NV];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const T *row = g + (size_t)__shfl_sync(0xffffffffU, mine, (q + u) & 31) * dim + col0;
#pragma unroll
                    for (int j = 0; j < NV; ++j) {
                        if (q + u < here && col0 + (lane + 32 * j) * VE < dim) v[u][j] = *reinterpret_cast<const vec *>(row + (lane + 32 * j) * VE);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (q + u < here) add_row(q + u, v[u]);
                }
            }
        }
    }
    __syncwarp();
    const bool goes_on = some && after == current;
    if (lane == 0) {
        first_token[warp] = begin;
        ends[warp] = some ? (token_before == begin ? 1U : 0U) | (goes_on ? 2U : 0U) | (token_before == begin && after == begin ? 4U : 0U) : 8U;
    }
    if (some) {
        if (goes_on && !open_left) keep(tail(warp)); else finish();
    }
    __syncthreads();
    // runs that cross the warps of the block, a thread per column, warps in order
    const unsigned c = min((unsigned)threadIdx.x, (unsigned)COLS - 1U);
    const bool column = threadIdx.x < COLS && col0 + c < dim;
    float sum = 0.0f, first = 0.0f;                            // of the run being added; of the one that began in an earlier piece
    bool from_before = true, open = false, closes = false;     // sum is still that one's; goes on behind the last warp; that one ends here
#pragma unroll
    for (int k = 0; k < ES_WARPS; ++k) {
        const unsigned f = ends[k];
        if (f & 8U) continue;
        open = (f & 2U) != 0U;
        if (f & 1U) {
            sum += head[k][c];
            if (!(f & 4U)) {
                if (from_before) {
                    closes = true;
                    first = sum;
                } else if (column) {
                    es_store<T, 1>(table + (size_t)first_token[k] * dim + col0 + c, &sum, scale, add);
                }
                sum = 0.0f;
            }
        }
        if (!(f & 4U)) {
            from_before = false;
            if (f & 2U) sum = tail(k)[c];
        }
    }
    if (open) {
        if (column) __stcg(&partial[((size_t)chunk * 2U + (from_before ? 0U : 1U)) * dim + col0 + c], sum);
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            atomicExch(&flags[(size_t)chunk * slabs + slab], 1U);
        }
    }
    if (!closes) return;
    // the piece in which the run begins: the one in front of the first piece whose preceding entry has the token
    const int tok = first_token[0];
    unsigned begins = chunk, full;   // (32 pieces looked at together, by every warp)
    do {
        const bool same = begins > (unsigned)lane + 1U && __ldg(&token[(size_t)(begins - 1U - lane) * piece - 1U]) == tok;
        const unsigned apart = ~__ballot_sync(0xffffffffU, same);
        full = apart != 0U ? (unsigned)__ffs((int)apart) - 1U : 32U;
        begins -= full;
    } while (full == 32U);
    begins -= 1U;
    for (unsigned k = begins + threadIdx.x; k < chunk; k += ES_WARPS * 32) {
        const unsigned *flag = &flags[(size_t)k * slabs + slab];
        unsigned polls = 0;
        while (es_load_acquire(flag) == 0U) {
            if (++polls == ES_POLLS) {
                atomicExch(err_flag, 611);
                break;
            }
        }
    }
    __syncthreads();
    if (!column) return;
    const float *part = partial + col0 + c;
    sum = __ldcg(part + ((size_t)begins * 2U + 1U) * dim);
#pragma unroll 16
    for (unsigned k = begins + 1U; k < chunk; ++k) sum += __ldcg(part + (size_t)k * 2U * dim);
    sum += first;
    es_store<T, 1>(table + (size_t)tok * dim + col0 + c, &sum, scale, add);
}

template <typename T, typename V>
gd_status lookup(gd_backend *be, const void *table, const int *ids, void *out, const gd_backend_embedding_args *a, float scale)
{
    const size_t vecs = a->dim / (sizeof(V) / sizeof(T));
#define GO(LANES)                                                                                                                                             \
    gdb_launch(es_lookup_kernel<T, V, LANES>, gdb_grid_for((a->ids_count + 4U * (256 / LANES) - 1U) / (4U * (256 / LANES)), 1U, be, 32U), 256, 0, be->stream, \
               (const V *)table, ids, (V *)out, a->ids_count, a->vocab, vecs, scale)
    if (vecs <= 16U) GO(16); else if (vecs <= 32U) GO(32); else if (vecs <= 64U) GO(64); else if (vecs <= 128U) GO(128); else GO(256);
#undef GO
    return gdb_launched(be, "embedding_scaled_forward");
}

template <typename T, int VE, int NV>
gd_status reduce(gd_backend *be, const void *g, const unsigned *order, const int *token, unsigned *count, void *table, float *partial, unsigned *flags, unsigned n, unsigned piece,
                 unsigned pieces, unsigned slabs, size_t dim, float scale, bool add)
{
    gdb_launch(es_reduce_kernel<T, VE, NV>, pieces * slabs, ES_WARPS * 32, 0, be->stream, (const T *)g, order, token, count, (T *)table, partial, flags, n, piece, slabs, dim, scale, add,
               be->err_flag);
    return gdb_launched(be, "embedding_sorted_backward sums");
}

template <typename T>
gd_status backward(gd_backend *be, const void *g, const int *ids, void *table, const gd_backend_embedding_args *a, float scale, bool add)
{
    constexpr int VE = sizeof(T) == 2 ? 8 : 4;
    const unsigned n = (unsigned)a->ids_count, vocab = (unsigned)a->vocab;
    const size_t dim = a->dim, row_bytes = dim * sizeof(T);
    const bool vec = dim % VE == 0U && (((uintptr_t)g | (uintptr_t)table) % 16U) == 0U;
    const size_t slabs = vec ? (dim + 32U * VE - 1U) / (32U * VE) : (dim + 255U) / 256U;
    // order, token, count and turns, partial sums, flags
    const size_t list = ((size_t)n * 4U + 255U) & ~(size_t)255U;
    if (2U * list + 256U + 2U * dim * sizeof(float) + slabs * sizeof(unsigned) > be->ws_bytes) return GD_ERR_OUT_OF_MEMORY;
    unsigned *order = reinterpret_cast<unsigned *>(be->ws);
    int *token = reinterpret_cast<int *>(be->ws + list);
    unsigned *count = reinterpret_cast<unsigned *>(be->ws + 2U * list);
    float *partial = reinterpret_cast<float *>(be->ws + 2U * list + 256U);
    const size_t fit = (be->ws_bytes - 2U * list - 256U) / (2U * dim * sizeof(float) + slabs * sizeof(unsigned));
    // entries of a warp: what gives every place on the GPU one block, 8 at least (rows on their way); more where the partial sums would not
    // fit the workspace
    const unsigned sms = gdb_usable_sms(be);
    size_t per = ((size_t)n * slabs + (size_t)sms * ES_BLOCKS * ES_WARPS - 1U) / ((size_t)sms * ES_BLOCKS * ES_WARPS);
    if (per < 8U) per = 8U;
    if (per > 4096U) per = 4096U;
    while (((size_t)n + per * ES_WARPS - 1U) / (per * ES_WARPS) > fit) per *= 2U;
    const size_t piece = per * ES_WARPS, pieces = ((size_t)n + piece - 1U) / piece;
    if (pieces * slabs > 0x7fffffffU) return GD_ERR_UNSUPPORTED;
    unsigned *flags = reinterpret_cast<unsigned *>(partial + pieces * 2U * dim);
    const unsigned n_flags = (unsigned)(pieces * slabs);
    // a slice of the vocabulary per block, two blocks' worth of SMs at most where the counters allow it
    unsigned width = (vocab + sms - 1U) / sms;
    if (width > ES_MAX_WIDTH) width = ES_MAX_WIDTH;
    const unsigned slices = (vocab + width - 1U) / width;
    // (more than half of an SM's shared memory: blocks that start while the preceding kernel drains would pair up on the SMs it left first)
    const unsigned range = ((n + ES_SORT_WARPS * 32U - 1U) / (ES_SORT_WARPS * 32U)) * 32U, room = (unsigned)((ES_SORT_SMEM - width * ES_SORT_WARPS * 4U) / (ES_SORT_WARPS * 8U));
    const unsigned notes = range < room ? range : room;
    int smem = (int)((width * 4U + notes * 8U) * ES_SORT_WARPS);
    if (smem < 116 * 1024) smem = 116 * 1024;
    static bool ready = false;
    if (!ready) {
        const int most = (int)ES_SORT_SMEM;
        cudaError_t e = cudaFuncSetAttribute(es_sort_kernel<uint4>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(es_sort_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return gdb_fail(be, e, "embedding_sorted_backward smem attribute");
        ready = true;
    }
    if (vec) {
        gdb_launch(es_sort_kernel<uint4>, slices, ES_SORT_WARPS * 32, smem, be->stream, ids, n, vocab, width, notes, order, token, count, flags, n_flags, add ? (uint4 *)nullptr : (uint4 *)table, row_bytes / 16U);
    } else {
        gdb_launch(es_sort_kernel<T>, slices, ES_SORT_WARPS * 32, smem, be->stream, ids, n, vocab, width, notes, order, token, count, flags, n_flags, add ? (T *)nullptr : (T *)table, dim);
    }
    gd_status st = gdb_launched(be, "embedding_sorted_backward sort");
    if (st != GD_OK) return st;
    return vec ? reduce<T, VE, 1>(be, g, order, token, count, table, partial, flags, n, (unsigned)piece, (unsigned)pieces, (unsigned)slabs, dim, scale, add)
               : reduce<T, 1, 8>(be, g, order, token, count, table, partial, flags, n, (unsigned)piece, (unsigned)pieces, (unsigned)slabs, dim, scale, add);
}

bool es_args_ok(const gd_backend_tensor_view *rows, const gd_backend_tensor_view *ids, const gd_backend_tensor_view *table, const gd_backend_embedding_args *a)
{
    return rows != NULL && ids != NULL && table != NULL && a != NULL && a->vocab > 0U && a->dim > 0U && a->vocab <= SIZE_MAX / 8U / a->dim &&
           a->ids_count <= SIZE_MAX / 8U / a->dim && rows->dtype == table->dtype && table->count == a->vocab * a->dim && ids->count == a->ids_count &&
           rows->count == a->ids_count * a->dim;
}

}  // namespace

extern "C" {

gd_status gdb200_embedding_scaled_forward(gd_backend *be, const gd_backend_tensor_view *table, const gd_backend_tensor_view *ids, const gd_backend_tensor_view *out, float scale,
                                          const gd_backend_embedding_args *args)
{
    if (be == NULL || !es_args_ok(out, ids, table, args)) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    const uint32_t dt = table->dtype;
    if (!gdb_is_float_dtype(dt)) {
        return GD_ERR_UNSUPPORTED;
    }
    const void *tp = gdb_tv_ptr(table, dt);
    const int *ip = (const int *)gdb_tv_ptr(ids, GDB_DTYPE_I32);
    void *op = gdb_tv_ptr(out, dt);
    if (tp == NULL || ip == NULL || op == NULL) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (args->ids_count == 0U) {
        return GD_OK;
    }
    const bool vec = args->dim % (16U / gdb_dtype_size(dt)) == 0U && (((uintptr_t)tp | (uintptr_t)op) % 16U) == 0U;
    if (dt == GDB_DTYPE_F16) return vec ? lookup<__half, uint4>(be, tp, ip, op, args, scale) : lookup<__half, __half>(be, tp, ip, op, args, scale);
    if (dt == GDB_DTYPE_BF16) return vec ? lookup<__nv_bfloat16, uint4>(be, tp, ip, op, args, scale) : lookup<__nv_bfloat16, __nv_bfloat16>(be, tp, ip, op, args, scale);
    return vec ? lookup<float, uint4>(be, tp, ip, op, args, scale) : lookup<float, float>(be, tp, ip, op, args, scale);
}

gd_status gdb200_embedding_sorted_backward(gd_backend *be, const gd_backend_tensor_view *grad_out, const gd_backend_tensor_view *ids, const gd_backend_tensor_view *grad_table,
                                           int32_t accumulate, float scale, const gd_backend_embedding_args *args)
{
    if (be == NULL || !es_args_ok(grad_out, ids, grad_table, args)) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    const uint32_t dt = grad_table->dtype;
    if (!gdb_is_float_dtype(dt) || args->ids_count > 0x7fffffffU || args->vocab > 0x7fffffffU) {
        return GD_ERR_UNSUPPORTED;
    }
    const void *gp = gdb_tv_ptr(grad_out, dt);
    const int *ip = (const int *)gdb_tv_ptr(ids, GDB_DTYPE_I32);
    void *tp = gdb_tv_ptr(grad_table, dt);
    if (gp == NULL || ip == NULL || tp == NULL) {
        return GD_ERR_INVALID_ARGUMENT;
    }
    if (args->ids_count == 0U) {
        if (accumulate != 0) return GD_OK;
        const cudaError_t e = cudaMemsetAsync(tp, 0, grad_table->count * gdb_dtype_size(dt), be->stream);
        be->launches += 1U;
        return e == cudaSuccess ? GD_OK : gdb_fail(be, e, "embedding_sorted_backward zero");
    }
    return dt == GDB_DTYPE_F16    ? backward<__half>(be, gp, ip, tp, args, scale, accumulate != 0)
           : dt == GDB_DTYPE_BF16 ? backward<__nv_bfloat16>(be, gp, ip, tp, args, scale, accumulate != 0)
                                  : backward<float>(be, gp, ip, tp, args, scale, accumulate != 0);
}

}  // extern "C"
