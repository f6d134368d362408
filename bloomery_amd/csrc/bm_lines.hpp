// What the products over codes share (8-bit integers, microscaled 4-bit floating point): the entries of experts' runs, their columns and outputs,
// and 128-byte lines of k on their way through LDS. A is a kernel's arguments: order, start, n_slots, top_k, n_cols, n_experts, rows, y, ld, et, fault
// and layer as the kernels name them.
#ifndef BM_LINES_HPP
#define BM_LINES_HPP

#include "bm_elem.hpp"

namespace bmk {

typedef int v4i __attribute__((ext_vector_type(4)));

// A dimension of a launch has fewer than 2^32 threads. Workgroups that would be more go along a second one, 2^20 a step; group_index numbers them through
// (the last step may be ragged: what it has too many finds nothing to do).
constexpr u32 kGroupsLog = 20;
static dim3 group_grid(uint64_t groups, u32 threads) {
    if (groups * threads <= 0xffffffffu) return dim3((u32)groups);
    return dim3(1u << kGroupsLog, (u32)((groups + (1u << kGroupsLog) - 1) >> kGroupsLog));
}
__device__ __forceinline__ u32 group_index() { return blockIdx.y << kGroupsLog | blockIdx.x; }

// Entry j's column; one that names no column raises ExpertId and gets column 0 with a NaN scale.
template <class A>
__device__ __forceinline__ u32 run_column(const A &a, u32 j, bool &bad) {
    bad = false;
    if (!a.order) return j;
    const u32 s = a.order[j], c = a.top_k ? s / a.top_k : j;
    if (s < a.n_slots && c < a.n_cols) return c;
    bad = true;
    return 0;
}

// The columns of N entries, their slots asked for at once.
template <int N, class A>
__device__ __forceinline__ void run_columns(const A &a, u32 (&j)[N]) {
    u32 s[N];
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = a.order[j[i]];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const u32 c = a.top_k ? s[i] / a.top_k : j[i];
        j[i] = s[i] < a.n_slots && c < a.n_cols ? c : 0u;
    }
}

// Four neighbouring values of an output row from r on, those below `rows`.
template <class A>
__device__ __forceinline__ void run_store4(const A &a, u32 j, u32 r, const float (&v)[4]) {
    const size_t at = (size_t)j * a.ld + r;
    const u32 have = a.rows - r;
    if (a.et == kElemF32) elem_store_some<kElemF32, 4>(a.y, at, have, v);
    else if (a.et == kElemF16) elem_store_some<kElemF16, 4>(a.y, at, have, v);
    else elem_store_some<kElemBF16, 4>(a.y, at, have, v);
}

// ---- lines through LDS. 128-byte lines of k, eight 16-byte pieces each, come from memory straight into LDS (16 bytes a lane, no register in between),
// eight lanes a line: asked for in the matrix instructions' own form, sixteen rows side by side in neighbouring lanes, a line would take the
// vector cache four times as long. Piece c of line r lies at place c ^ swizzle(r), which the lane that asks for it arranges, so that the
// pieces that the matrix instructions take of 16 lines at once come from all the banks.
typedef __attribute__((address_space(1))) void lds_from;
typedef __attribute__((address_space(3))) void lds_to;

// An instruction's 16-byte reads are served for lanes 0..3, 12..15, 20..27 at once, then for 4..11, 16..19, 28..31, and so on from 32: sixteen lanes of two
// neighbouring groups of sixteen lines, which have different pieces. So lines 0..3 and 12..15 have the turns 0..3, the others 4..7: the two groups' reads meet no bank twice if both pieces
// are among a line's first four or both among its last four, as line_piece's and mx4_of_line's are (pieces 0 and 4 would meet every bank twice). (With (line >> 1) & 7 pieces that differ by 2 met
// every bank twice: 30 % of the time of the 4-bit product of 4096 x 7168 x 7168. The 8-bit products, whose pieces differ by 1, take the same time with both.)
__device__ __forceinline__ u32 line_swizzle(u32 line) { return ((line >> 1) ^ (line & 4)) & 7; }

// N groups of eight lines of a wave's own, a stage of its ring. Line l of rows that end before the piece does is read at its first
// piece, which is there; whoever multiplies puts zeros in the columns' place.
template <int N>
struct Lines {
    static constexpr int kStage = N * 1024;
    const int8_t *from[N]; // this lane's row of each group
    u32 piece[2];          // and its piece, of even and odd groups
    __device__ __forceinline__ void begin(u32 lane) {
#pragma unroll
        for (u32 g = 0; g < 2; g++) piece[g] = 16 * ((lane & 7) ^ line_swizzle(8 * g + (lane >> 3)));
    }
    __device__ __forceinline__ void ask(uint8_t *stage, u32 line, u32 kp) const {
        u32 at[2];
#pragma unroll
        for (int g = 0; g < 2; g++) at[g] = 128 * line + (128 * line + piece[g] < kp ? piece[g] : 0u);
#pragma unroll
        for (int g = 0; g < N; g++) __builtin_amdgcn_global_load_lds((lds_from *)(from[g] + at[g & 1]), (lds_to *)(stage + g * 1024), 16, 0, 0);
    }
};
// What the matrix instructions take of line group t (sixteen lines) of a stage: half c of the lines.
__device__ __forceinline__ v4i line_piece(const uint8_t *stage, u32 lane, int t, int c) {
    return *reinterpret_cast<const v4i *>(stage + t * 2048 + (lane & 15) * 128 + 16 * ((4 * c + (lane >> 4)) ^ line_swizzle(lane & 15)));
}
// All but the last n of a wave's loads have landed, and its reads are done.
template <int n>
__device__ __forceinline__ void loads_landed() {
    static_assert(n < 64, "vmcnt");
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | (n >> 4) << 14); // vmcnt(n) lgkmcnt(0)
    __asm__ volatile("" ::: "memory");
}

// The workgroup's writes to LDS are there for all of it; loads on their way into LDS are not waited for.
__device__ __forceinline__ void lds_meet() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// A tile of the experts: their runs cut into tiles of BT entries, numbered through the experts in order. False: there is none of that number. The bounds
// of 256 experts are asked for at once; a run that is none has no tiles. `check`: every run is looked at, those behind the tile too, and one that
// is none raises ExpertId (one workgroup of a launch does so).
template <int BT, class A>
__device__ __forceinline__ bool run_tile(const A &a, u32 tile, bool check, u32 &expert, u32 &t0) {
    const u32 lane = threadIdx.x & 63;
    u32 before = 0;
    bool found = false;
    for (u32 e0 = 0; e0 < a.n_experts; e0 += 256) {
        u32 j0[4], j1[4];
#pragma unroll
        for (u32 i = 0; i < 4; i++) {
            const u32 e = min(e0 + 64 * i + lane, a.n_experts - 1);
            j0[i] = a.start[e];
            j1[i] = a.start[e + 1];
        }
        if (check) {
            bool none = false;
#pragma unroll
            for (u32 i = 0; i < 4; i++) none |= j0[i] > j1[i] || j1[i] > a.n_slots; // (lanes past the last look at the last once more)
            if (none) bm_raise(a.fault, a.layer, kSiteExpertId);
            if (found) continue;
        }
#pragma unroll
        for (u32 i = 0; i < 4; i++) {
            const u32 e = e0 + 64 * i + lane;
            if (e0 + 64 * i >= a.n_experts) break;
            const bool run = j0[i] <= j1[i] && j1[i] <= a.n_slots;
            const u32 c = e < a.n_experts && run ? (j1[i] - j0[i] + BT - 1) / BT : 0;
            u32 upto = c;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const u32 o = (u32)__shfl_up((int)upto, d, 64);
                if (lane >= (u32)d) upto += o;
            }
            const unsigned long long mine = __ballot(c != 0 && before + upto - c <= tile && tile < before + upto);
            if (mine) {
                const int l = __builtin_ctzll(mine);
                expert = (u32)__builtin_amdgcn_readfirstlane((int)(e0 + 64 * i + (u32)l));
                t0 = (u32)__builtin_amdgcn_readfirstlane((int)((tile - before - (u32)__shfl((int)(upto - c), l, 64)) * BT));
                if (!check) return true;
                found = true;
                break;
            }
            before += (u32)__shfl((int)upto, 63, 64);
        }
    }
    return found;
}

// ---- tiles of columns and rows. G: a tile's kColumns, kRows, kWaves, kStage, RR (a wave's loads of rows a step) and kUp.

// The eight rows of a wave's r-th load: where there are not as many for every wave, the last ones are asked for again.
template <class G>
__device__ __forceinline__ u32 tile_row_group(u32 wave, int r) {
    const u32 group = wave * G::RR + r;
    return G::kRows % (8 * G::kWaves) == 0 ? group : min(group, (u32)G::kRows / 8 - 1);
}

// Where a lane's reads begin, for each 64 bytes of a step: of rows and of columns. The upper buffers' carry the first one's place with them
// (and are read that far in front), so that a read's address is one register and a constant that its instruction can hold.
struct TileAt {
    u32 a[2], b[2];
};
// What the matrix instructions take of 64 bytes of k of N tiles, from the FIRST on.
template <class G, int B, int N>
__device__ __forceinline__ void tile_read(v4i (&f)[N], const uint8_t *__restrict__ buf, u32 at, int first) {
    constexpr u32 up = B >= G::kUp ? (u32)G::kUp * G::kStage : 0u;
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = *reinterpret_cast<const v4i *>(buf + (int)(at - up + (first + i) * 2048));
}

// READS of what comes next between MFMAS products of what is there.
template <int READS, int MFMAS>
__device__ __forceinline__ void tile_weave() {
#pragma unroll
    for (int i = 0; i < READS; i++) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);              // an LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, MFMAS / READS ? MFMAS / READS : 1, 0); // products
    }
}

// Where piece p of column c lies in a line of LINE pieces: turned by the column within the pieces' largest power of two.
template <int LINE>
__device__ __forceinline__ u32 tile_turned(u32 p, u32 c) {
    constexpr u32 kPow = LINE & -LINE;
    return p ^ (c & (kPow - 1));
}

} // namespace bmk

#endif // BM_LINES_HPP
