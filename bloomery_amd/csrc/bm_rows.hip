// Tokens' rows sorted by expert and back, for experts that are computed by other means than this library's GGUF kernels: the
// tables of a router's picks, the rows moved behind them, the weighted sum onto the residual, and the gradients of both.
//
//   order, start   bm_buckets' (crates/gpu/src/q4k_sel.rs:20-41): the listed slots by expert, ascending inside a run
//   place[s]       where slot s stands in order, 0xffffffff for a slot that no run lists: order's inverse, which lets every
//                  row be written (and every sum be formed) by a workgroup that owns it, without atomics
//
// Everything here moves memory: a token's row is read once and stored at its slots' places, a sum's rows are read once and
// asked for together. Rates below count every byte once, read or written, on MI355X, where a copy of 1 GiB runs at 5.2 TB/s.
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

// A token's row to the places of its slots in LDS (kUnlisted: not stored). EB: bytes of an element. The row's first pieces are asked for before
// the places are known (row_ahead): the two latencies run side by side.
template <u32 N>
struct RowAhead {
    uint4 v[N];
};
template <u32 N>
__device__ __forceinline__ RowAhead<N> row_ahead(const SortArgs &a, u32 token, u32 thread, u32 threads) {
    RowAhead<N> r;
    const uint8_t *from = a.x + (size_t)token * a.x_line;
#pragma unroll
    for (u32 i = 0; i < N; i++) {
        const u32 at = 16 * (thread + i * threads);
        if (at + 16 <= a.row_bytes) r.v[i] = bm_ld16u(from + at);
    }
    return r;
}
// (eight threads at least)
template <int EB, u32 N>
__device__ __forceinline__ void move_row(const SortArgs &a, u32 token, const u32 *places, const RowAhead<N> &ahead, u32 thread, u32 threads) {
    const uint8_t *from = a.x + (size_t)token * a.x_line;
    const auto piece = [&](u32 at, uint4 v) {
        for (u32 k = 0; k < a.top_k; k++)
            if (places[k] != kUnlisted) __builtin_memcpy(a.rows + (size_t)places[k] * a.rows_line + at, &v, 16);
    };
#pragma unroll
    for (u32 i = 0; i < N; i++) {
        const u32 at = 16 * (thread + i * threads);
        if (at + 16 <= a.row_bytes) piece(at, ahead.v[i]);
    }
    for (u32 at = 16 * (thread + N * threads); at + 16 <= a.row_bytes; at += 16 * threads) piece(at, bm_ld16u(from + at));
    // what is left of a row that is no whole number of pieces, an element a thread
    const u32 b = (a.row_bytes & ~15u) + EB * thread;
    if (b < a.row_bytes)
        for (u32 k = 0; k < a.top_k; k++)
            if (places[k] != kUnlisted) __builtin_memcpy(a.rows + (size_t)places[k] * a.rows_line + b, from + b, EB);
}

// The whole sort in one launch: a workgroup takes T tokens (as many as make eight slots, or one) and finds its slots' places by counting what stands in
// front of them among all the slots (a comparison a slot and id, the wave's answers counted by the scalar unit), and one more workgroup
// finds the runs' bounds. Work grows with the square of the slots, so it is for few of them; what bounds it is the launch, then the counting.
// us, this / three launches: 128 slots 4.7 / 9.7, 1024 5.2 / 10.3, 2048 6.6 / 11.0, 4096 10.3 / 12.1, 6144 14.2 / 13.2 (rows of 2048 bf16, eight slots a token);
// 4096 tokens of one slot 9.5 / 11.3 (a workgroup a token: 19.5).
template <int EB, u32 T>
__global__ __launch_bounds__(kRowThreads) void k_sort_few(SortArgs a) {
    __shared__ u32 places[T == 1 ? kMaxCombineSlots : 8];
    __shared__ u32 count[kBucketExperts], scan[kRowThreads];
    const u32 n = a.n_tokens * a.top_k, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (blockIdx.x == gridDim.x - 1) { // the bounds: counts, then their running sum, four experts a thread
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
    const u32 token = blockIdx.x * T, s0 = token * a.top_k, have = min(T, a.n_tokens - token) * a.top_k;
    RowAhead<T == 1 ? 2 : 1> ahead[T];
    if (a.x)
#pragma unroll
        for (u32 t = 0; t < T; t++) ahead[t] = row_ahead<T == 1 ? 2 : 1>(a, min(token + t, a.n_tokens - 1), tid, kRowThreads);
    for (u32 k = tid; k < have; k += kRowThreads) places[k] = 0;
    __syncthreads();
    for (u32 k0 = 0; k0 < have; k0 += 8) {
        u32 mine[8], before[8];
        for (u32 k = 0; k < 8; k++) {
            const u32 s = s0 + (k0 + k < have ? k0 + k : k0);
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
                if (k0 + k < have) atomicAdd(&places[k0 + k], before[k]);
    }
    __syncthreads();
    for (u32 k = tid; k < have; k += kRowThreads) {
        const bool listed = a.sel[s0 + k] < a.n_experts;
        const u32 p = listed ? places[k] : kUnlisted;
        places[k] = p;
        a.place[s0 + k] = p;
        if (listed) a.order[p] = s0 + k;
    }
    if (!a.x) return;
    __syncthreads();
#pragma unroll
    for (u32 t = 0; t < T; t++)
        if (token + t < a.n_tokens) move_row<EB>(a, token + t, places + t * a.top_k, ahead[t], tid, kRowThreads);
}
template <int EB>
static void few_launch(const Launch &L, const SortArgs &a) {
    const auto start = [&](auto kernel, u32 tokens) { hipLaunchKernelGGL(kernel, dim3((a.n_tokens + tokens - 1) / tokens + 1), dim3(kRowThreads), 0, L.stream, a); };
    if (a.top_k > 4) start(k_sort_few<EB, 1>, 1);
    else if (a.top_k > 2) start(k_sort_few<EB, 2>, 2);
    else if (a.top_k == 2) start(k_sort_few<EB, 4>, 4);
    else start(k_sort_few<EB, 8>, 8);
}

// ---- many slots, in three launches over chunks of slots, a wave each.
// 1. A chunk's counts an expert into work[chunk * n_experts + expert], and every slot's rank among its chunk's slots of its expert into
//    place. Eight waves share a chunk, an eighth each with counts of its own: the slots of a wave that share an expert find each other bit
//    by bit of the id, and an expert's counts are summed over the waves in front. (One wave a chunk of 512 took 6.2 us where this takes 4.)
constexpr u32 kSortWaves = 8;
__host__ __device__ inline u32 sort_chunk_len(u32 n) {
    const u32 per = (n + 255) / 256, least = 64 * kSortWaves; // at most 256 chunks
    return (per + least - 1) / least * least;
}

__global__ __launch_bounds__(64 * kSortWaves) void k_sort_count(SortArgs a, u32 n, u32 per) {
    __shared__ u32 count[kSortWaves * kBucketExperts];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, share = per / kSortWaves;
    const u32 lo = blockIdx.x * per + wave * share, hi = min(lo + share, n);
    u32 id = lo + lane < hi ? a.sel[lo + lane] : kUnlisted; // the first 64 slots' ids come while the counts are cleared
    for (u32 i = tid; i < kSortWaves * a.n_experts; i += 64 * kSortWaves) count[i] = 0;
    __syncthreads();
    u32 *mine = count + wave * a.n_experts;
    const int bits = 32 - __builtin_clz(a.n_experts | 1u);
    u32 first = 0; // the rank of the only slot a lane has where a wave has 64 at most
    for (u32 b = lo; b < hi; b += 64) {
        const u32 s = b + lane;
        if (b != lo) id = s < hi ? a.sel[s] : kUnlisted;
        const bool listed = id < a.n_experts;
        if (!listed && id != kUnlisted) bm_raise(a.fault, a.layer, kSiteExpertId);
        unsigned long long same = __ballot(listed);
        for (int k = 0; k < bits; k++) {
            const unsigned long long set = __ballot((id >> k) & 1u);
            same &= ((id >> k) & 1u) ? set : ~set;
        }
        const u32 below = (u32)__builtin_popcountll(same & ((1ull << lane) - 1ull));
        const u32 had = listed ? mine[id] : 0; // every lane of the wave reads before the first of a group adds
        if (listed && below == 0) mine[id] = had + (u32)__builtin_popcountll(same);
        first = had + below;
        if (share > 64 && s < hi) a.place[s] = first;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    for (u32 e = tid; e < a.n_experts; e += 64 * kSortWaves) { // counts -> what the waves in front hold
        u32 sum = 0;
#pragma unroll
        for (u32 w = 0; w < kSortWaves; w++) {
            const u32 c = count[w * a.n_experts + e];
            count[w * a.n_experts + e] = sum;
            sum += c;
        }
        a.work[(size_t)blockIdx.x * a.n_experts + e] = sum;
    }
    __syncthreads();
    for (u32 b = lo; b < hi; b += 64) {
        const u32 s = b + lane;
        if (s >= hi) break;
        if (share > 64) id = a.sel[s], first = a.place[s];
        a.place[s] = id < a.n_experts ? mine[id] + first : kUnlisted;
    }
}

// 2. The counts become the places of the chunks' first slots (4 us for 64 chunks of 128 experts, latency: one workgroup, two passes): running sums over an expert's chunks behind the runs' bounds. A thread has an expert
//    and a run of the chunks (at most 32 threads an expert), whose counts it asks for sixteen at a time; it keeps the first sixteen, and reads what
//    is behind them twice, the second time from the cache.
__global__ __launch_bounds__(1024) void k_sort_scan(SortArgs a, u32 chunks, u32 log_experts) {
    __shared__ u32 part[1024], scan[16];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u32 e = tid & ((1u << log_experts) - 1u), group = tid >> log_experts, groups = min(1024u >> log_experts, 32u);
    const u32 share = (chunks + groups - 1) / groups, lo = min(group * share, chunks), hi = e < a.n_experts ? min(lo + share, chunks) : lo;
    u32 sum = 0, first[16];
    const auto counts = [&](u32 c0, u32 (&v)[16]) {
#pragma unroll
        for (u32 i = 0; i < 16; i++) v[i] = c0 + i < hi ? a.work[(size_t)(c0 + i) * a.n_experts + e] : 0;
    };
    counts(lo, first);
#pragma unroll
    for (u32 i = 0; i < 16; i++) sum += first[i];
    for (u32 c0 = lo + 16; c0 < hi; c0 += 16) {
        u32 v[16];
        counts(c0, v);
#pragma unroll
        for (u32 i = 0; i < 16; i++) sum += v[i];
    }
    part[tid] = sum;
    __syncthreads();
    u32 before = 0, count = 0; // of this expert: in the groups in front, in all
    for (u32 g = 0; g < groups; g++) {
        const u32 v = part[(g << log_experts) + e];
        before += g < group ? v : 0;
        count += v;
    }
    // the bounds: the running sum over the experts, in the first group's threads
    const u32 c = group == 0 ? count : 0;
    u32 upto = c;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u32 o = (u32)__shfl_up((int)upto, d, 64);
        if (lane >= (u32)d) upto += o;
    }
    if (lane == 63) scan[wave] = upto;
    __syncthreads(); // (every thread has read its part)
    u32 at = upto - c;
#pragma unroll
    for (u32 w = 0; w < 16; w++) at += w < wave ? scan[w] : 0;
    if (group == 0) part[e] = at;
    __syncthreads();
    if (group == 0 && e < a.n_experts) {
        a.start[e] = at;
        if (e + 1 == a.n_experts) a.start[a.n_experts] = at + count;
    }
    at = part[e] + before;
    const auto settle = [&](u32 c0, const u32 (&v)[16]) {
#pragma unroll
        for (u32 i = 0; i < 16; i++) {
            if (c0 + i < hi) a.work[(size_t)(c0 + i) * a.n_experts + e] = at;
            at += v[i];
        }
    };
    settle(lo, first);
    for (u32 c0 = lo + 16; c0 < hi; c0 += 16) {
        u32 v[16];
        counts(c0, v);
        settle(c0, v);
    }
}

// 3. Places and order of a token's slots, and its row to them. Memory: 4096 tokens of 2048 bf16 to eight places each, 151 MB, in 27 to 31 us, 4.9 to 5.6 TB/s.
__device__ __forceinline__ u32 sort_settle(const SortArgs &a, u32 s, u32 per) {
    const u32 id = a.sel[s], rank = a.place[s];
    if (id >= a.n_experts) return kUnlisted; // place holds kUnlisted already
    const u32 p = a.work[(size_t)(s / per) * a.n_experts + id] + rank;
    a.place[s] = p;
    a.order[p] = s;
    return p;
}
//    1 << log threads a token, several tokens a workgroup where rows are short (the whole sort, three launches, of 4810 tokens, eight slots, 128 wide, 13.4 us; a workgroup a token 15.6).
template <int EB>
__global__ __launch_bounds__(kRowThreads) void k_sort_move(SortArgs a, u32 per, u32 log) {
    __shared__ u32 places[kRowThreads / 8 * kMaxCombineSlots];
    const u32 tid = threadIdx.x, mine = tid >> log, thread = tid & ((1u << log) - 1u), tokens = kRowThreads >> log;
    const u32 token0 = blockIdx.x * tokens, token = min(token0 + mine, a.n_tokens - 1), have = min(tokens, a.n_tokens - token0) * a.top_k;
    const RowAhead<2> ahead = row_ahead<2>(a, token, thread, 1u << log);
    for (u32 i = tid; i < have; i += kRowThreads) places[i] = sort_settle(a, token0 * a.top_k + i, per);
    __syncthreads();
    if (token0 + mine < a.n_tokens) move_row<EB>(a, token, places + mine * a.top_k, ahead, thread, 1u << log);
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
        if (eb == 4) few_launch<4>(L, a);
        else few_launch<2>(L, a);
        return hipGetLastError();
    }
    const u32 per = sort_chunk_len(n), chunks = (n + per - 1) / per;
    hipLaunchKernelGGL(k_sort_count, dim3(chunks), dim3(64 * kSortWaves), 0, L.stream, a, n, per);
    u32 log_experts = 0;
    while ((1u << log_experts) < a.n_experts) log_experts++;
    hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, L.stream, a, chunks, log_experts);
    if (!x) hipLaunchKernelGGL(k_sort_places, dim3((n + kRowThreads - 1) / kRowThreads), dim3(kRowThreads), 0, L.stream, a, n, per);
    else {
        u32 log = 3;
        while (log < 8 && (16u << log) < a.row_bytes) log++;
        const u32 tokens = kRowThreads >> log;
        const dim3 grid((a.n_tokens + tokens - 1) / tokens);
        if (eb == 4) hipLaunchKernelGGL(k_sort_move<4>, grid, dim3(kRowThreads), 0, L.stream, a, per, log);
        else hipLaunchKernelGGL(k_sort_move<2>, grid, dim3(kRowThreads), 0, L.stream, a, per, log);
    }
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

// A batch of K slots' places and weights. A slot that is not listed (or past the token's last) is read through the place of one that is, or the
// first row, and what comes is not used: its request is answered by the cache, and no branch parts the batch.
template <int K>
struct Slots {
    u32 p[K];
    float w[K];
    bool on[K];
};
template <int K>
__device__ __forceinline__ Slots<K> slots_of(const u32 *place, const float *w, size_t s0, u32 have, u32 n_slots, u32 *fault, u32 layer) {
    Slots<K> r;
#pragma unroll
    for (u32 k = 0; k < K; k++) {
        const size_t s = s0 + (k < have ? k : 0);
        r.p[k] = k < have ? place[s] : kUnlisted;
        r.w[k] = w ? w[s] : 1.0f;
    }
    u32 some = 0;
#pragma unroll
    for (u32 k = 0; k < K; k++) {
        r.p[k] = checked_place(r.p[k], n_slots, fault, layer);
        r.on[k] = r.p[k] != kUnlisted;
        some = r.on[k] ? r.p[k] : some;
    }
#pragma unroll
    for (u32 k = 0; k < K; k++) r.p[k] = r.on[k] ? r.p[k] : some;
    return r;
}

// y[t] = (acc = 0; slots ascending: acc = fma(w, row, acc)) + resid[t], in f32 and rounded once: bm_combine_tokens' order. A thread holds a
// 16-byte piece of a token (1 << log threads a token, several tokens a workgroup where rows are short); its slots' rows are asked for eight
// at a time, so that a row's latency is paid once for all of them. What is left of a row that is no whole number of pieces goes an element a thread.
// Memory: 1500 tokens of 7168 f16 from eight rows each, 194 MB, in 41.5 us, 4.7 TB/s; 16 tokens 4.9 us, the launch.
template <int ET, int K>
__device__ __forceinline__ void combine_piece(const CombineArgs &a, const Slots<K> &s, u32 c, float (&acc)[kElemPiece<ET>]) {
    uint4 v[K];
#pragma unroll
    for (u32 k = 0; k < K; k++) v[k] = elem_piece<ET>(a.rows, (size_t)s.p[k] * a.ld_rows + c);
#pragma unroll
    for (u32 k = 0; k < K; k++) {
        float f[kElemPiece<ET>];
        elem_unpack<ET>(v[k], f);
#pragma unroll
        for (int j = 0; j < kElemPiece<ET>; j++) acc[j] = s.on[k] ? fmaf(s.w[k], f[j], acc[j]) : acc[j];
    }
}
template <int ET, int K, bool ALL> // ALL: at most K slots a token, whose places a thread keeps
__global__ __launch_bounds__(kRowThreads) void k_expert_combine(CombineArgs a, u32 log) {
    constexpr int V = kElemPiece<ET>;
    const u32 t = blockIdx.x * (kRowThreads >> log) + (threadIdx.x >> log), mine = threadIdx.x & ((1u << log) - 1u);
    if (t >= a.n_tokens) return;
    const size_t s0 = (size_t)t * a.top_k;
    Slots<K> s;
    if constexpr (ALL) s = slots_of<K>(a.place, a.w, s0, a.top_k, a.n_slots, a.fault, a.layer);
    for (u32 c = V * mine; c + V <= a.width; c += V << log) {
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = 0.0f;
        uint4 r;
        if (a.resid) r = elem_piece<ET>(a.resid, (size_t)t * a.ld_resid + c);
        if constexpr (ALL) {
            combine_piece<ET, K>(a, s, c, acc);
        } else {
            for (u32 k0 = 0; k0 < a.top_k; k0 += K) {
                s = slots_of<K>(a.place, a.w, s0 + k0, a.top_k - k0, a.n_slots, a.fault, a.layer);
                combine_piece<ET, K>(a, s, c, acc);
            }
        }
        if (a.resid) {
            float f[V];
            elem_unpack<ET>(r, f);
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] = __fadd_rn(acc[j], f[j]);
        }
        elem_piece_store<ET>(a.y, (size_t)t * a.ld_y + c, elem_pack<ET>(acc));
    }
    const u32 c = a.width / V * V + mine; // (1 << log is V at least)
    if (c >= a.width) return;
    float acc = 0.0f;
    for (u32 k = 0; k < a.top_k; k++) {
        const u32 p = checked_place(a.place[s0 + k], a.n_slots, a.fault, a.layer);
        if (p != kUnlisted) acc = fmaf(a.w ? a.w[s0 + k] : 1.0f, elem_load1<ET>(a.rows, (size_t)p * a.ld_rows + c), acc);
    }
    if (a.resid) acc = __fadd_rn(acc, elem_load1<ET>(a.resid, (size_t)t * a.ld_resid + c));
    elem_store1<ET>(a.y, (size_t)t * a.ld_y + c, acc);
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

// d_rows[place[s]] = w[s] dy[t], d_w[s] = <dy[t], rows[place[s]]>: T threads a token (the workgroup, or a wave where rows are short), K slots at a time, so
// that a piece of dy is read once for K rows that are asked for together. Every dot is summed in one order: a thread's pieces, the wave, the
// four waves. Memory, as much read as written: 4096 tokens of 2048 bf16, 285 MB, in 60 us, 4.7 TB/s.
template <int ET, int K, int T>
__global__ __launch_bounds__(kRowThreads) void k_expert_combine_grad(CombineGradArgs a) {
    constexpr int V = kElemPiece<ET>;
    __shared__ float part[4][K];
    const u32 t = blockIdx.x * (kRowThreads / T) + threadIdx.x / T, tid = threadIdx.x % T;
    if (t >= a.n_tokens) return; // whole waves (T = 64), or nobody
    for (u32 k0 = 0; k0 < a.top_k; k0 += K) {
        const Slots<K> s = slots_of<K>(a.place, a.w, (size_t)t * a.top_k + k0, a.top_k - k0, a.n_slots, a.fault, a.layer);
        float dot[K] = {};
        for (u32 c = V * tid; c + V <= a.width; c += V * T) {
            uint4 v[K];
            const uint4 gp = elem_piece<ET>(a.dy, (size_t)t * a.ld_dy + c);
#pragma unroll
            for (u32 k = 0; k < K; k++) v[k] = elem_piece<ET>(a.rows, (size_t)s.p[k] * a.ld_rows + c);
            float g[V];
            elem_unpack<ET>(gp, g);
#pragma unroll
            for (u32 k = 0; k < K; k++) {
                float f[V], d[V];
                elem_unpack<ET>(v[k], f);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    dot[k] = fmaf(g[j], f[j], dot[k]);
                    d[j] = __fmul_rn(s.w[k], g[j]);
                }
                if (s.on[k]) elem_piece_store<ET>(a.d_rows, (size_t)s.p[k] * a.ld_d_rows + c, elem_pack<ET>(d));
            }
        }
        const u32 c = a.width / V * V + tid;
        if (c < a.width) {
            const float g = elem_load1<ET>(a.dy, (size_t)t * a.ld_dy + c);
#pragma unroll
            for (u32 k = 0; k < K; k++)
                if (s.on[k]) {
                    dot[k] = fmaf(g, elem_load1<ET>(a.rows, (size_t)s.p[k] * a.ld_rows + c), dot[k]);
                    elem_store1<ET>(a.d_rows, (size_t)s.p[k] * a.ld_d_rows + c, __fmul_rn(s.w[k], g));
                }
        }
#pragma unroll
        for (u32 k = 0; k < K; k++) {
            const float sum = wave_sum(s.on[k] ? dot[k] : 0.0f);
            if constexpr (T == 64) {
                if (tid == 0 && k0 + k < a.top_k) a.d_w[(size_t)t * a.top_k + k0 + k] = sum;
            } else if ((tid & 63) == 0) {
                part[tid >> 6][k] = sum;
            }
        }
        if constexpr (T > 64) {
            __syncthreads();
            if (tid < K && k0 + tid < a.top_k)
                a.d_w[(size_t)t * a.top_k + k0 + tid] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
            __syncthreads();
        }
    }
}

template <int ET>
static void combine_launch(const Launch &L, const CombineArgs &a) {
    const u32 pieces = a.width / kElemPiece<ET>;
    u32 log = 3;
    while (log < 8 && (1u << log) < pieces) log++;
    const u32 tokens = kRowThreads >> log;
    const dim3 grid((a.n_tokens + tokens - 1) / tokens), block(kRowThreads);
    if (a.top_k == 1) hipLaunchKernelGGL((k_expert_combine<ET, 1, true>), grid, block, 0, L.stream, a, log);
    else if (a.top_k == 2) hipLaunchKernelGGL((k_expert_combine<ET, 2, true>), grid, block, 0, L.stream, a, log);
    else if (a.top_k <= 4) hipLaunchKernelGGL((k_expert_combine<ET, 4, true>), grid, block, 0, L.stream, a, log);
    else if (a.top_k <= 8) hipLaunchKernelGGL((k_expert_combine<ET, 8, true>), grid, block, 0, L.stream, a, log);
    else hipLaunchKernelGGL((k_expert_combine<ET, 8, false>), grid, block, 0, L.stream, a, log);
}

// us, bf16. A batch as small as the token's slots, which eight at a time would ask for again: 4096 tokens of one slot, 2048 wide, gradients 9.8 (by eights 20.3), sum 6.1 (12.7); of
// four 24.6 and 14.4 (29.5, 17.3). A wave a token up to 128 pieces: 4096 tokens of eight slots, 1024 wide, 25.1 (a workgroup a token 29.3), 8192 tokens, 512 wide, 25.7
// (41.0), of two slots 8.1 (32.8); 1400 wide by workgroups 31.
template <int ET, int K>
static void grad_start(const Launch &L, const CombineGradArgs &a) {
    const dim3 block(kRowThreads);
    if (a.width <= 128 * kElemPiece<ET>) hipLaunchKernelGGL((k_expert_combine_grad<ET, K, 64>), dim3((a.n_tokens + 3) / 4), block, 0, L.stream, a);
    else hipLaunchKernelGGL((k_expert_combine_grad<ET, K, 256>), dim3(a.n_tokens), block, 0, L.stream, a);
}
template <int ET>
static void grad_launch(const Launch &L, const CombineGradArgs &a) {
    if (a.top_k == 1) grad_start<ET, 1>(L, a);
    else if (a.top_k == 2) grad_start<ET, 2>(L, a);
    else if (a.top_k <= 4) grad_start<ET, 4>(L, a);
    else grad_start<ET, 8>(L, a);
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
    if (et == kElemF32) grad_launch<kElemF32>(L, a);
    else if (et == kElemF16) grad_launch<kElemF16>(L, a);
    else grad_launch<kElemBF16>(L, a);
    return hipGetLastError();
}

} // namespace bmk
