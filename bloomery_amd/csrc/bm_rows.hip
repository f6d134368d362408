// Tokens' rows sorted by expert and back, for experts that are computed by other means than this library's GGUF kernels: the
// tables of a router's picks, the rows moved behind them, the weighted sum onto the residual, and the gradients of both.
//
//   order, start   bm_buckets' (crates/gpu/src/q4k_sel.rs:20-41): the listed slots by expert, ascending inside a run
//   place[s]       where slot s stands in order, 0xffffffff for a slot that no run lists: order's inverse, which lets every
//                  row be written (and every sum be formed) by a workgroup that owns it, without atomics
//
// Everything here moves memory: a token's row is read once and stored at its slots' places, a sum's rows are read once and
// asked for together.
#include "bm_elem.hpp"

namespace bmk {

constexpr u32 kUnlisted = 0xffffffffu; // the host's slot id, and the place of a slot that joins no run
constexpr u32 kRowThreads = 256;

// Slots and ids as one word each, so that one comparison counts what stands in front of a slot: a smaller expert, or the same
// and a smaller slot. 1024 experts x 2^22 slots fill 32 bits; an unlisted slot's word is below none.
__device__ __forceinline__ u32 sort_key(u32 id, u32 n_experts, u32 slot) { return id < n_experts ? (id << kTileExpertShift) | slot : 0xffffffffu; }

struct SortArgs {
    const u32 *sel;
    u32 n_tokens, top_k, n_experts;
    const uint8_t *x;
    size_t x_line; // bytes between two rows
    uint8_t *rows;
    size_t rows_line;
    u32 row_bytes;
    u32 *order, *start, *place, *work;
    u32 *fault, layer;
};

// A token's row to the places of its slots in LDS (kUnlisted: not stored). EB: bytes of an element.
template <int EB>
__device__ __forceinline__ void move_row(const SortArgs &a, u32 token, const u32 *places) {
    const uint8_t *from = a.x + (size_t)token * a.x_line;
    for (u32 at = 16 * threadIdx.x; at < a.row_bytes; at += 16 * kRowThreads) {
        if (at + 16 <= a.row_bytes) {
            const uint4 v = bm_ld16u(from + at);
            for (u32 k = 0; k < a.top_k; k++)
                if (places[k] != kUnlisted) __builtin_memcpy(a.rows + (size_t)places[k] * a.rows_line + at, &v, 16);
        } else {
            for (u32 b = at; b < a.row_bytes; b += EB)
                for (u32 k = 0; k < a.top_k; k++)
                    if (places[k] != kUnlisted) __builtin_memcpy(a.rows + (size_t)places[k] * a.rows_line + b, from + b, EB);
        }
    }
}

// The whole sort in one launch: a workgroup a token finds its slots' places by counting what stands in front of them among all
// the slots (a comparison a slot and id, the wave's answers counted by the scalar unit), and one more workgroup finds the runs'
// bounds. Work grows with tokens x slots, so it is for few of them.
template <int EB>
__global__ __launch_bounds__(kRowThreads) void k_sort_few(SortArgs a) {
    __shared__ u32 places[kMaxCombineSlots];
    __shared__ u32 count[kBucketExperts], scan[kRowThreads];
    const u32 n = a.n_tokens * a.top_k, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (blockIdx.x == a.n_tokens) { // the bounds: counts, then their running sum, four experts a thread
        for (u32 e = tid; e < kBucketExperts; e += kRowThreads) count[e] = 0;
        __syncthreads();
        for (u32 s = tid; s < n; s += kRowThreads) {
            const u32 id = a.sel[s];
            if (id < a.n_experts) atomicAdd(&count[id], 1u);
            else if (id != kUnlisted) bm_raise(a.fault, a.layer, kSiteExpertId);
        }
        __syncthreads();
        u32 c[4], sum = 0;
        for (int i = 0; i < 4; i++) c[i] = count[4 * tid + i], sum += c[i];
        scan[tid] = sum;
        __syncthreads();
        for (u32 d = 1; d < kRowThreads; d <<= 1) {
            const u32 below = tid >= d ? scan[tid - d] : 0;
            __syncthreads();
            scan[tid] += below;
            __syncthreads();
        }
        u32 at = scan[tid] - sum;
        for (u32 i = 0; i < 4; i++) {
            const u32 e = 4 * tid + i;
            if (e < a.n_experts) a.start[e] = at;
            at += c[i];
            if (e + 1 == a.n_experts) a.start[a.n_experts] = at;
        }
        return;
    }
    const u32 token = blockIdx.x, s0 = token * a.top_k;
    for (u32 k = tid; k < a.top_k; k += kRowThreads) places[k] = 0;
    __syncthreads();
    for (u32 k0 = 0; k0 < a.top_k; k0 += 8) {
        u32 mine[8], before[8];
        for (u32 k = 0; k < 8; k++) {
            const u32 s = s0 + (k0 + k < a.top_k ? k0 + k : k0);
            mine[k] = sort_key(a.sel[s], a.n_experts, s);
            before[k] = 0;
        }
        for (u32 b = 64 * wave; b < n; b += kRowThreads) {
            const u32 s = b + lane, key = s < n ? sort_key(a.sel[s], a.n_experts, s) : 0xffffffffu;
#pragma unroll
            for (u32 k = 0; k < 8; k++) before[k] += (u32)__builtin_popcountll(__ballot(key < mine[k]));
        }
        if (lane == 0)
#pragma unroll
            for (u32 k = 0; k < 8; k++)
                if (k0 + k < a.top_k) atomicAdd(&places[k0 + k], before[k]);
    }
    __syncthreads();
    for (u32 k = tid; k < a.top_k; k += kRowThreads) {
        const bool listed = a.sel[s0 + k] < a.n_experts;
        const u32 p = listed ? places[k] : kUnlisted;
        places[k] = p;
        a.place[s0 + k] = p;
        if (listed) a.order[p] = s0 + k;
    }
    if (!a.x) return;
    __syncthreads();
    move_row<EB>(a, token, places);
}

// ---- many slots, in three launches over chunks of slots, a wave each.
// 1. A chunk's counts an expert into work[chunk * n_experts ..], and every slot's rank among its chunk's slots of its expert into
//    place (the slots of a wave that share an expert find each other bit by bit of the id).
__host__ __device__ inline u32 sort_chunk_len(u32 n) {
    const u32 per = (n + 255) / 256; // at most 256 chunks
    return per < 512 ? 512 : (per + 63) & ~63u;
}

__global__ __launch_bounds__(64) void k_sort_count(SortArgs a, u32 n, u32 per) {
    __shared__ u32 count[kBucketExperts];
    const u32 lane = threadIdx.x, lo = blockIdx.x * per, hi = lo + per < n ? lo + per : n;
    for (u32 e = lane; e < a.n_experts; e += 64) count[e] = 0;
    __syncthreads();
    const int bits = 32 - __builtin_clz(a.n_experts | 1u);
    for (u32 b = lo; b < hi; b += 64) {
        const u32 s = b + lane, id = s < hi ? a.sel[s] : kUnlisted;
        const bool listed = id < a.n_experts;
        if (!listed && id != kUnlisted) bm_raise(a.fault, a.layer, kSiteExpertId);
        unsigned long long same = __ballot(listed);
        for (int k = 0; k < bits; k++) {
            const unsigned long long set = __ballot((id >> k) & 1u);
            same &= ((id >> k) & 1u) ? set : ~set;
        }
        const u32 below = (u32)__builtin_popcountll(same & ((1ull << lane) - 1ull));
        const u32 had = listed ? count[id] : 0; // every lane of the wave reads before the first of a group adds
        if (listed && below == 0) count[id] = had + (u32)__builtin_popcountll(same);
        if (s < hi) a.place[s] = listed ? had + below : kUnlisted;
        __syncthreads();
    }
    for (u32 e = lane; e < a.n_experts; e += 64) a.work[(size_t)blockIdx.x * a.n_experts + e] = count[e];
}

// 2. The counts' running sums over chunks inside an expert, behind the experts' own: work becomes the place of a chunk's first slot.
__global__ __launch_bounds__(1024) void k_sort_scan(SortArgs a, u32 chunks) {
    __shared__ u32 scan[17];
    const u32 e = threadIdx.x;
    u32 sum = 0;
    if (e < a.n_experts)
        for (u32 c = 0; c < chunks; c++) sum += a.work[(size_t)c * a.n_experts + e];
    u32 total;
    u32 at = block_scan_1024(sum, scan, &total);
    if (e < a.n_experts) {
        a.start[e] = at;
        for (u32 c = 0; c < chunks; c++) {
            const u32 v = a.work[(size_t)c * a.n_experts + e];
            a.work[(size_t)c * a.n_experts + e] = at;
            at += v;
        }
    }
    if (e == 0) a.start[a.n_experts] = total;
}

// 3. Places and order of a token's slots, and its row to them.
__device__ __forceinline__ u32 sort_settle(const SortArgs &a, u32 s, u32 per) {
    const u32 id = a.sel[s];
    if (id >= a.n_experts) return kUnlisted; // place holds kUnlisted already
    const u32 p = a.work[(size_t)(s / per) * a.n_experts + id] + a.place[s];
    a.place[s] = p;
    a.order[p] = s;
    return p;
}
template <int EB>
__global__ __launch_bounds__(kRowThreads) void k_sort_move(SortArgs a, u32 per) {
    __shared__ u32 places[kMaxCombineSlots];
    const u32 token = blockIdx.x;
    if (threadIdx.x < a.top_k) places[threadIdx.x] = sort_settle(a, token * a.top_k + threadIdx.x, per);
    __syncthreads();
    move_row<EB>(a, token, places);
}
__global__ __launch_bounds__(kRowThreads) void k_sort_places(SortArgs a, u32 n, u32 per) {
    const u32 s = blockIdx.x * kRowThreads + threadIdx.x;
    if (s < n) sort_settle(a, s, per);
}

size_t expert_sort_work(int n_slots, int n_experts) {
    if ((u32)n_slots <= kSortFew) return 0;
    const u32 per = sort_chunk_len((u32)n_slots);
    return (size_t)(((u32)n_slots + per - 1) / per) * (size_t)n_experts;
}

hipError_t expert_sort(const Launch &L, const uint32_t *sel, int n_tokens, int top_k, int n_experts, const void *x, int et, int64_t ldx,
                       int width, uint32_t *order, uint32_t *start, uint32_t *place, void *rows, int64_t ld_rows, uint32_t *work) {
    const int eb = elem_bytes(et);
    const u32 n = (u32)n_tokens * (u32)top_k;
    const SortArgs a = {sel, (u32)n_tokens, (u32)top_k, (u32)n_experts, static_cast<const uint8_t *>(x), (size_t)ldx * eb,
                        static_cast<uint8_t *>(rows), (size_t)ld_rows * eb, (u32)width * (u32)eb, order, start, place, work, L.fault, L.layer};
    if (n <= kSortFew) {
        if (eb == 4) hipLaunchKernelGGL(k_sort_few<4>, dim3((unsigned)n_tokens + 1), dim3(kRowThreads), 0, L.stream, a);
        else hipLaunchKernelGGL(k_sort_few<2>, dim3((unsigned)n_tokens + 1), dim3(kRowThreads), 0, L.stream, a);
        return hipGetLastError();
    }
    const u32 per = sort_chunk_len(n), chunks = (n + per - 1) / per;
    hipLaunchKernelGGL(k_sort_count, dim3(chunks), dim3(64), 0, L.stream, a, n, per);
    hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, L.stream, a, chunks);
    if (!x) hipLaunchKernelGGL(k_sort_places, dim3((n + kRowThreads - 1) / kRowThreads), dim3(kRowThreads), 0, L.stream, a, n, per);
    else if (eb == 4) hipLaunchKernelGGL(k_sort_move<4>, dim3((unsigned)n_tokens), dim3(kRowThreads), 0, L.stream, a, per);
    else hipLaunchKernelGGL(k_sort_move<2>, dim3((unsigned)n_tokens), dim3(kRowThreads), 0, L.stream, a, per);
    return hipGetLastError();
}

// --------------------------------------------------------------------------------------- sums and gradients

struct CombineArgs {
    const void *rows; // the experts' rows, by place
    size_t ld_rows;
    const u32 *place;
    const float *w;    // NULL: ones
    const void *resid; // NULL: none
    size_t ld_resid;
    void *y;
    size_t ld_y;
    u32 n_tokens, top_k, width, n_slots;
    u32 *fault, layer;
};

// A slot's place as it may be read through: kUnlisted for one that is not listed, and for one past the rows, which raises ExpertId.
__device__ __forceinline__ u32 checked_place(u32 p, u32 n_slots, u32 *fault, u32 layer) {
    if (p < n_slots) return p;
    if (p != kUnlisted) bm_raise(fault, layer, kSiteExpertId);
    return kUnlisted;
}

// y[t] = (acc = 0; slots ascending: acc = fma(w, row, acc)) + resid[t], in f32 and rounded once: bm_combine_tokens' order. A thread holds
// eight values of a token (1 << log threads a token, several tokens a workgroup where rows are short); its slots' places, weights
// and rows are asked for eight slots at a time, so that a row's latency is paid once for all of them.
template <int ET>
__global__ __launch_bounds__(kRowThreads) void k_expert_combine(CombineArgs a, u32 log) {
    const u32 t = blockIdx.x * (kRowThreads >> log) + (threadIdx.x >> log);
    if (t >= a.n_tokens) return;
    for (u32 c = 8 * (threadIdx.x & ((1u << log) - 1u)); c < a.width; c += 8u << log) {
        const u32 have = a.width - c;
        float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (a.resid) elem_load_some<ET, 8>(a.resid, (size_t)t * a.ld_resid + c, have, r);
        for (u32 k0 = 0; k0 < a.top_k; k0 += 8) {
            u32 p[8];
            float w[8], v[8][8];
#pragma unroll
            for (u32 k = 0; k < 8; k++) {
                const u32 s = t * a.top_k + (k0 + k < a.top_k ? k0 + k : k0);
                p[k] = k0 + k < a.top_k ? a.place[s] : kUnlisted;
                w[k] = a.w ? a.w[s] : 1.0f;
            }
#pragma unroll
            for (u32 k = 0; k < 8; k++) {
                p[k] = checked_place(p[k], a.n_slots, a.fault, a.layer);
                if (p[k] != kUnlisted) elem_load_some<ET, 8>(a.rows, (size_t)p[k] * a.ld_rows + c, have, v[k]);
                else
#pragma unroll
                    for (int j = 0; j < 8; j++) v[k][j] = 0.0f;
            }
#pragma unroll
            for (u32 k = 0; k < 8; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) acc[j] = p[k] != kUnlisted ? fmaf(w[k], v[k][j], acc[j]) : acc[j];
        }
        if (a.resid)
#pragma unroll
            for (int j = 0; j < 8; j++) acc[j] = __fadd_rn(acc[j], r[j]);
        elem_store_some<ET, 8>(a.y, (size_t)t * a.ld_y + c, have, acc);
    }
}

struct CombineGradArgs {
    const void *dy;
    size_t ld_dy;
    const void *rows;
    size_t ld_rows;
    const u32 *place;
    const float *w;
    void *d_rows;
    size_t ld_d_rows;
    float *d_w;
    u32 n_tokens, top_k, width, n_slots;
    u32 *fault, layer;
};

// d_rows[place[s]] = w[s] dy[t], d_w[s] = <dy[t], rows[place[s]]>: a workgroup a token, eight slots at a time, so that a piece of dy is
// read once for eight rows that are asked for together. Every dot is summed in one order: a thread's pieces, the wave, the
// four waves.
template <int ET>
__global__ __launch_bounds__(kRowThreads) void k_expert_combine_grad(CombineGradArgs a) {
    __shared__ float part[4][8];
    const u32 t = blockIdx.x, tid = threadIdx.x;
    for (u32 k0 = 0; k0 < a.top_k; k0 += 8) {
        u32 p[8];
        float w[8], dot[8];
#pragma unroll
        for (u32 k = 0; k < 8; k++) {
            const u32 s = t * a.top_k + (k0 + k < a.top_k ? k0 + k : k0);
            p[k] = k0 + k < a.top_k ? checked_place(a.place[s], a.n_slots, a.fault, a.layer) : kUnlisted;
            w[k] = a.w[s];
            dot[k] = 0.0f;
        }
        for (u32 c = 8 * tid; c < a.width; c += 8 * kRowThreads) {
            const u32 have = a.width - c;
            float g[8], v[8][8];
            elem_load_some<ET, 8>(a.dy, (size_t)t * a.ld_dy + c, have, g);
#pragma unroll
            for (u32 k = 0; k < 8; k++)
                if (p[k] != kUnlisted) elem_load_some<ET, 8>(a.rows, (size_t)p[k] * a.ld_rows + c, have, v[k]);
#pragma unroll
            for (u32 k = 0; k < 8; k++)
                if (p[k] != kUnlisted) {
                    float d[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        dot[k] = fmaf(g[j], v[k][j], dot[k]);
                        d[j] = __fmul_rn(w[k], g[j]);
                    }
                    elem_store_some<ET, 8>(a.d_rows, (size_t)p[k] * a.ld_d_rows + c, have, d);
                }
        }
#pragma unroll
        for (u32 k = 0; k < 8; k++) {
            const float sum = wave_sum(dot[k]);
            if ((tid & 63) == 0) part[tid >> 6][k] = sum;
        }
        __syncthreads();
        if (tid < 8 && k0 + tid < a.top_k)
            a.d_w[(size_t)t * a.top_k + k0 + tid] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
        __syncthreads();
    }
}

template <int ET>
static void combine_launch(const Launch &L, const CombineArgs &a) {
    const u32 pieces = (a.width + 7) / 8;
    u32 log = 3;
    while (log < 8 && (1u << log) < pieces) log++;
    const u32 tokens = kRowThreads >> log;
    hipLaunchKernelGGL(k_expert_combine<ET>, dim3((a.n_tokens + tokens - 1) / tokens), dim3(kRowThreads), 0, L.stream, a, log);
}

hipError_t expert_combine(const Launch &L, const void *rows, int et, int64_t ld_rows, const uint32_t *place, const float *w, const void *resid,
                          int64_t ld_resid, int n_tokens, int top_k, int width, void *y, int64_t ld_y) {
    const CombineArgs a = {rows, (size_t)ld_rows, place, w, resid, (size_t)ld_resid, y, (size_t)ld_y, (u32)n_tokens, (u32)top_k, (u32)width,
                           (u32)n_tokens * (u32)top_k, L.fault, L.layer};
    if (et == kElemF32) combine_launch<kElemF32>(L, a);
    else if (et == kElemF16) combine_launch<kElemF16>(L, a);
    else combine_launch<kElemBF16>(L, a);
    return hipGetLastError();
}

hipError_t expert_combine_grad(const Launch &L, const void *dy, int et, int64_t ld_dy, const void *rows, int64_t ld_rows, const uint32_t *place,
                               const float *w, int n_tokens, int top_k, int width, void *d_rows, int64_t ld_d_rows, float *d_w) {
    const CombineGradArgs a = {dy, (size_t)ld_dy, rows, (size_t)ld_rows, place, w, d_rows, (size_t)ld_d_rows, d_w, (u32)n_tokens, (u32)top_k,
                               (u32)width, (u32)n_tokens * (u32)top_k, L.fault, L.layer};
    const dim3 grid((unsigned)n_tokens), block(kRowThreads);
    if (et == kElemF32) hipLaunchKernelGGL(k_expert_combine_grad<kElemF32>, grid, block, 0, L.stream, a);
    else if (et == kElemF16) hipLaunchKernelGGL(k_expert_combine_grad<kElemF16>, grid, block, 0, L.stream, a);
    else hipLaunchKernelGGL(k_expert_combine_grad<kElemBF16>, grid, block, 0, L.stream, a);
    return hipGetLastError();
}

} // namespace bmk
