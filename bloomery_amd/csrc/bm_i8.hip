// Matrix products in 8-bit integers: rows quantized with a scale each (a token's activations, or a matrix's channels), an exact
// int32 sum on the matrix cores, both scales on the way out. One matrix, or the matrices of experts over the runs of slots that a
// router made.
//
//   scale  s = f32(max |x| / 127)
//   code   q = the real quotient x / s rounded to the nearest whole number, halves to even, held to +-127
//   value  y = f32(sum of q w) * s_token * s_row, three f32 roundings, one more to the output's type
//
// A row of codes is k rounded up to 16 bytes, zeros behind the last value. The integer sum is exact for k up to 131072 (127 * 128 a product),
// so every split of k gives the same bits.
#include "bm_elem.hpp"

#include <algorithm>

namespace bmk {

typedef int v4i __attribute__((ext_vector_type(4)));

// A dimension of a launch has fewer than 2^32 threads. Workgroups that would be more go along a second one, 2^20 a step; i8_group numbers them through
// (the last step may be ragged: what it has too many finds nothing to do).
constexpr u32 kGroupsLog = 20;
static dim3 i8_grid(uint64_t groups, u32 threads) {
    if (groups * threads <= 0xffffffffu) return dim3((u32)groups);
    return dim3(1u << kGroupsLog, (u32)((groups + (1u << kGroupsLog) - 1) >> kGroupsLog));
}
__device__ __forceinline__ u32 i8_group() { return blockIdx.y << kGroupsLog | blockIdx.x; }

// ------------------------------------------------------------------------------------------------ quantizer

// The code of v under scale s (normal, not small), inv = fl(1 / s). rint(v * inv) is off by one at most, and only where the quotient lies
// within 127 * 2^-22 of a half; the remainder v - n s is exact there (v and n s are multiples of ulp(s) / 2 at least, their difference is
// below 2^24 of those), so comparing twice of it with s decides as the real quotient would.
__device__ __forceinline__ int i8_code(float v, float s, float inv) {
    float n = rintf(__fmul_rn(v, inv));
    const float rest = fmaf(-n, s, v), twice = 2.0f * fabsf(rest);
    const bool odd = ((int)n) & 1;
    if (twice > s || (twice == s && odd)) n += copysignf(1.0f, rest);
    return (int)fminf(fmaxf(n, -127.0f), 127.0f);
}

// A row's scale from the bits of its largest magnitude (positive floats order as their bits; infinities and NaN lie on top).
struct I8Scale {
    float s, up, su, inv; // small scales, whose reciprocal could overflow, go up by 2^100 with their values (exactly)
    bool bad, zero;
};
__device__ __forceinline__ I8Scale i8_scale(u32 most) {
    I8Scale r;
    r.bad = most >= 0x7f800000u;
    r.s = r.bad ? bm_bits_f32(0x7fc00000u) : __fdiv_rn(bm_bits_f32(most), 127.0f);
    r.up = r.s < 0x1p-64f ? 0x1p100f : 1.0f;
    r.su = r.s * r.up;
    r.inv = __fdiv_rn(1.0f, r.su);
    r.zero = r.bad || r.s == 0.0f;
    return r;
}
// The eight codes. fl(1 / s) is off by 2^-24 of itself, the product with v by 127 * 2^-24 at most: unless that product lies within 2^-16 of a half
// (three values in a hundred thousand), its nearest whole number is the quotient's, and one addition that leaves it in the low bits
// gives it: seven instructions a value where the exact form takes some twenty. Else the exact form.
__device__ __forceinline__ uint2 i8_codes(const float (&v)[8], const I8Scale &s) {
    if (s.zero) return make_uint2(0, 0);
    constexpr float kMagic = 12582912.0f;
    u32 t[8];
    bool near = s.up != 1.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float sum = fmaf(v[j], s.inv, kMagic), rest = fmaf(v[j], s.inv, -__fsub_rn(sum, kMagic));
        t[j] = bm_f32_bits(sum);
        near |= !(fabsf(rest) <= 0.5f - 0x1p-16f);
    }
    if (near)
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = (u32)i8_code(v[j] * s.up, s.su, s.inv);
    u32 word[2];
#pragma unroll
    for (int j = 0; j < 2; j++)
        word[j] = __builtin_amdgcn_perm(t[4 * j + 1], t[4 * j], 0x0c0c0400u) | __builtin_amdgcn_perm(t[4 * j + 3], t[4 * j + 2], 0x04000c0cu);
    return make_uint2(word[0], word[1]);
}

struct QuantArgs {
    const void *x, *u; // u: the second input of a gate rule
    size_t ld;
    u32 m, k, kp;
    const u32 *live; // rows at or past it stay as they are (NULL: all m)
    int8_t *codes;
    float *scales;
    GateRule rule;
    u32 *fault, layer;
};

template <int ET, bool GLU>
__device__ __forceinline__ void quant_values(const QuantArgs &a, u32 row, u32 c, float (&v)[8], bool &odd) {
    const u32 have = c < a.k ? a.k - c : 0;
    if (have == 0) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
        return;
    }
    elem_load_some<ET, 8>(a.x, (size_t)row * a.ld + c, have, v);
    if constexpr (GLU) {
        float u[8];
        elem_load_some<ET, 8>(a.u, (size_t)row * a.ld + c, have, u);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            bool o = false;
            v[j] = (u32)j < have ? bm_gate_rule(a.rule.act, a.rule.limit, v[j], u[j], o) : 0.0f;
            odd |= o;
        }
    }
}

// A thread's CH pieces of a row, from piece `first` on, T apart: whole pieces are all asked for before the first is looked at (a thread past the last asks
// for that one and takes zeros), the ragged one that a row may end with by itself.
template <int ET, bool GLU, int T, int CH>
struct QuantPieces {
    static constexpr int V = kElemPiece<ET>, P = 8 / V;
    uint4 x[CH][P], u[GLU ? CH : 1][P];
    __device__ __forceinline__ void ask(const QuantArgs &a, u32 row, u32 first) {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const size_t at = (size_t)row * a.ld + 8 * min(first + i * T, a.k / 8 - 1);
#pragma unroll
            for (int p = 0; p < P; p++) {
                x[i][p] = elem_piece<ET>(a.x, at + p * V);
                if constexpr (GLU) u[i][p] = elem_piece<ET>(a.u, at + p * V);
            }
        }
    }
    __device__ __forceinline__ void values(const QuantArgs &a, u32 row, u32 first, float (&v)[CH][8], bool &odd) const {
        const u32 whole = a.k / 8;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const bool in = first + i * T < whole;
#pragma unroll
            for (int p = 0; p < P; p++) {
                float e[V];
                elem_unpack<ET>(x[i][p], e);
                if constexpr (GLU) {
                    float f[V];
                    elem_unpack<ET>(u[i][p], f);
                    if (a.rule.act == 0u) { // a piece's values together, no branch between them
#pragma unroll
                        for (int j = 0; j < V; j++) e[j] = bm_swiglu(e[j], f[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < V; j++) {
                            bool o = false;
                            e[j] = bm_gate_rule(a.rule.act, a.rule.limit, in ? e[j] : 0.0f, in ? f[j] : 0.0f, o);
                            odd |= o;
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < V; j++) v[i][p * V + j] = in ? e[j] : 0.0f;
            }
        }
        if ((a.k & 7) && whole % T == first && whole / T < CH) {
            float tail[8];
            quant_values<ET, GLU>(a, row, 8 * whole, tail, odd);
#pragma unroll
            for (int i = 0; i < CH; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] = (u32)i == whole / T ? tail[j] : v[i][j];
        }
    }
};

// T threads a row (a wave, or the workgroup), CH pieces of eight values a thread held in registers between the maximum and the codes; CH = 0: a
// row of any length, read twice (the second time from the cache).
template <int ET, bool GLU, int T, int CH>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_i8_quantize(QuantArgs a) {
    constexpr int kThreads = T < 256 ? 256 : T;
    __shared__ u32 top[T / 64];
    const u32 lane = threadIdx.x % T, row = i8_group() * (kThreads / T) + threadIdx.x / T;
    const u32 m = a.live ? min(a.m, *a.live) : a.m;
    if (row >= m) return; // whole waves (T = 64) or the workgroup
    float v[CH ? CH : 1][8];
    u32 most = 0;
    bool odd = false;
    const u32 pieces = a.kp / 8;
    if constexpr (CH > 0) {
        QuantPieces<ET, GLU, T, CH> in;
        if (a.k >= 8) {
            in.ask(a, row, lane);
            in.values(a, row, lane, v, odd);
        } else {
#pragma unroll
            for (int i = 0; i < CH; i++) quant_values<ET, GLU>(a, row, 8 * (lane + i * T), v[i], odd);
        }
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) most = max(most, bm_f32_bits(v[i][j]) & 0x7fffffffu);
    } else {
        for (u32 c = lane; c < pieces; c += T) {
            quant_values<ET, GLU>(a, row, 8 * c, v[0], odd);
#pragma unroll
            for (int j = 0; j < 8; j++) most = max(most, bm_f32_bits(v[0][j]) & 0x7fffffffu);
        }
    }
    if (GLU && odd) bm_raise(a.fault, a.layer, kSiteF32Product);
    most = bm_max32(most);
    most = max(most, (u32)__shfl_xor((int)most, 32, 64));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < T / 64; w++) most = max(most, top[w]);
    }
    const I8Scale sc = i8_scale(most);
    if (lane == 0) {
        a.scales[row] = sc.s;
        if (sc.bad) bm_raise(a.fault, a.layer, kSiteQuantColumn);
    }
    int8_t *out = a.codes + (size_t)row * a.kp;
#pragma unroll
    for (int i = 0; i < (CH ? CH : 1); i++)
        for (u32 c = lane + (u32)i * T; c < pieces; c += CH ? pieces : T) {
            if constexpr (CH == 0) quant_values<ET, GLU>(a, row, 8 * c, v[0], odd);
            *reinterpret_cast<uint2 *>(out + 8 * c) = i8_codes(v[i], sc);
        }
}

template <int ET, bool GLU, int T, int CH>
static void quant_start(const Launch &L, const QuantArgs &a) {
    constexpr u32 threads = T < 256 ? 256 : T, rows = threads / T;
    hipLaunchKernelGGL((k_i8_quantize<ET, GLU, T, CH>), i8_grid((a.m + rows - 1) / rows, threads), dim3(threads), 0, L.stream, a);
}
// us on MI355X, bf16, alone and behind the gate rule. While the rows are not eight a compute unit a row's length is dealt to more threads, a piece each: 24 x
// 7168 4.0 and 4.2 (256 threads of four pieces: 5.5, 6.3), 1500 x 7168 10.2 and 15.2 (10.8, 16.7), 1024 x 4096 4.9 and 6.8 (5.4, 7.6); behind that more pieces a thread
// ask for more at once: 4096 x 7168 18.2 and 32.6 (1024 threads: 22.0, 34.7); 18.2 us are 4.8 TB/s, what a copy reaches. Short rows take a wave each, 16384 x 768 11.5
// and 19.0 (a workgroup: 16.2, 30.6). Rows past 8192 values are read twice, a piece in flight a thread, the rule's values formed twice: 4096 x 18432 56.4 and 151 (4.0 and 2.5
// TB/s), 256 x 18432 6.7 and 12.6, one row 5.2 and 10.6.
template <int ET, bool GLU>
static void quant_launch(const Launch &L, const QuantArgs &a) {
    const bool few = a.m <= 2048;
    if (a.kp <= 512) quant_start<ET, GLU, 64, 1>(L, a);
    else if (a.kp <= 1024) quant_start<ET, GLU, 64, 2>(L, a);
    else if (a.kp <= 2048) quant_start<ET, GLU, 256, 1>(L, a);
    else if (a.kp <= 4096) few ? quant_start<ET, GLU, 512, 1>(L, a) : quant_start<ET, GLU, 256, 2>(L, a);
    else if (a.kp <= 8192) few ? quant_start<ET, GLU, 1024, 1>(L, a) : quant_start<ET, GLU, 256, 4>(L, a);
    else quant_start<ET, GLU, 1024, 0>(L, a);
}

hipError_t i8_quantize(const Launch &L, const void *x, const void *u, int et, int64_t ld, int m, int k, const uint32_t *live, int8_t *codes,
                       float *scales) {
    const QuantArgs a = {x, u, (size_t)ld, (u32)m, (u32)k, (u32)i8_row_bytes(k), live, codes, scales, L.rule, L.fault, L.layer};
    if (u) {
        if (et == kElemF32) quant_launch<kElemF32, true>(L, a);
        else if (et == kElemF16) quant_launch<kElemF16, true>(L, a);
        else quant_launch<kElemBF16, true>(L, a);
    } else {
        if (et == kElemF32) quant_launch<kElemF32, false>(L, a);
        else if (et == kElemF16) quant_launch<kElemF16, false>(L, a);
        else quant_launch<kElemBF16, false>(L, a);
    }
    return hipGetLastError();
}

// -------------------------------------------------------------------------------------------------- product

struct I8Args {
    const int8_t *w; // rows (of one matrix, or of an expert's) x kp
    const float *ws;
    u32 rows, kp;
    const int8_t *q; // columns x kp
    const float *qs;
    u32 m;             // columns of one matrix's product
    const u32 *order;  // experts: entry j's slot (NULL: entry j reads column j)
    const u32 *start;  // experts' runs (NULL: one matrix)
    u32 n_slots, top_k, n_cols, n_experts;
    void *y;
    size_t ld;
    int et;
    u32 *fault, layer;
};

// A run of entries and the matrix they meet.
struct I8Run {
    u32 j0, j1;
    const int8_t *w;
    const float *ws;
};
__device__ __forceinline__ bool i8_run(const I8Args &a, u32 e, I8Run &r) {
    if (!a.start) {
        r = I8Run{0, a.m, a.w, a.ws};
        return true;
    }
    const u32 j0 = a.start[e], j1 = a.start[e + 1];
    if (j0 > j1 || j1 > a.n_slots) { // no run of a table over these slots
        if (threadIdx.x == 0) bm_raise(a.fault, a.layer, kSiteExpertId);
        return false;
    }
    r = I8Run{j0, j1, a.w + (size_t)e * a.rows * a.kp, a.ws + (size_t)e * a.rows};
    return j1 > j0;
}
// Entry j's column; one that names no column raises ExpertId and gets column 0 with a NaN scale.
__device__ __forceinline__ u32 i8_column(const I8Args &a, u32 j, bool &bad) {
    bad = false;
    if (!a.order) return j;
    const u32 s = a.order[j], c = a.top_k ? s / a.top_k : j;
    if (s < a.n_slots && c < a.n_cols) return c;
    bad = true;
    return 0;
}

// The columns of N entries, their slots asked for at once.
template <int N>
__device__ __forceinline__ void i8_columns(const I8Args &a, u32 (&j)[N]) {
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
__device__ __forceinline__ void i8_store4(const I8Args &a, u32 j, u32 r, const float (&v)[4]) {
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
typedef __attribute__((address_space(1))) void i8_gptr;
typedef __attribute__((address_space(3))) void i8_lptr;

__device__ __forceinline__ u32 i8_swizzle(u32 line) { return (line >> 1) & 7; }

// N groups of eight lines of a wave's own, a stage of its ring. Line l of rows that end before the piece does is read at its first
// piece, which is there; whoever multiplies puts zeros in the columns' place.
template <int N>
struct I8Lines {
    static constexpr int kStage = N * 1024;
    const int8_t *from[N]; // this lane's row of each group
    u32 piece[2];          // and its piece, of even and odd groups
    __device__ __forceinline__ void begin(u32 lane) {
#pragma unroll
        for (u32 g = 0; g < 2; g++) piece[g] = 16 * ((lane & 7) ^ i8_swizzle(8 * g + (lane >> 3)));
    }
    __device__ __forceinline__ void ask(uint8_t *stage, u32 line, u32 kp) const {
        u32 at[2];
#pragma unroll
        for (int g = 0; g < 2; g++) at[g] = 128 * line + (128 * line + piece[g] < kp ? piece[g] : 0u);
#pragma unroll
        for (int g = 0; g < N; g++) __builtin_amdgcn_global_load_lds((i8_gptr *)(from[g] + at[g & 1]), (i8_lptr *)(stage + g * 1024), 16, 0, 0);
    }
};
// What the matrix instructions take of line group t (sixteen lines) of a stage: half c of the lines.
__device__ __forceinline__ v4i i8_of_line(const uint8_t *stage, u32 lane, int t, int c) {
    return *reinterpret_cast<const v4i *>(stage + t * 2048 + (lane & 15) * 128 + 16 * ((4 * c + (lane >> 4)) ^ i8_swizzle(lane & 15)));
}
// All but the last n of a wave's loads have landed, and its reads are done.
template <int n>
__device__ __forceinline__ void i8_landed() {
    static_assert(n < 64, "vmcnt");
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | (n >> 4) << 14); // vmcnt(n) lgkmcnt(0)
    __asm__ volatile("" ::: "memory");
}

// The workgroup's writes to LDS are there for all of it; loads on their way into LDS are not waited for.
__device__ __forceinline__ void i8_meet() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// Few columns a matrix, bound by the launch and by a line's way from memory (24 x 7168 x 2048: 14.7 MB of weights in 5.1 us, 2.9 TB/s; 7168 x 7168 and one column: 51 MB
// in 9.6, 5.3 TB/s): 16 R rows a workgroup against 16 C columns, its NW waves dealing the row's lines among them, each through a ring of four
// stages of its own, two on their way while one is multiplied and the fourth is asked for. The waves' sums meet in LDS as integers.
template <int R, int C, int NW>
__global__ __launch_bounds__(64 * NW) void k_i8_few(I8Args a) {
    typedef I8Lines<2 * (R + C)> L;
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], ring2[NW * L::kStage], ring3[NW * L::kStage];
    static_assert(R * C * 1024 <= L::kStage && R * C <= NW, "a wave's sums lie in its stage, one piece a thread");
    const u32 lane = threadIdx.x & 63, tid = threadIdx.x, wave = (u32)__builtin_amdgcn_readfirstlane(tid >> 6);
    I8Run run;
    if (!i8_run(a, blockIdx.y, run)) return;
    const u32 r0 = blockIdx.x * (16 * R), lines = (a.kp + 127) / 128, mine = wave * L::kStage;
    L src;
    src.begin(lane);
#pragma unroll
    for (u32 g = 0; g < 2 * R; g++) src.from[g] = run.w + (size_t)min(r0 + 8 * g + (lane >> 3), a.rows - 1) * a.kp; // rows past the last are not stored
    for (u32 t0 = run.j0 + blockIdx.z * (16 * C); t0 < run.j1; t0 += gridDim.z * (16 * C)) {
        u32 col[2 * C];
#pragma unroll
        for (u32 g = 0; g < 2 * C; g++) col[g] = min(t0 + 8 * g + (lane >> 3), run.j1 - 1);
        if (a.order) i8_columns<2 * C>(a, col);
#pragma unroll
        for (u32 g = 0; g < 2 * C; g++) src.from[2 * R + g] = a.q + (size_t)col[g] * a.kp;
        if (wave < lines) src.ask(ring0 + mine, wave, a.kp);
        if (wave + NW < lines) src.ask(ring1 + mine, wave + NW, a.kp);
        if (wave + 2 * NW < lines) src.ask(ring2 + mine, wave + 2 * NW, a.kp);
        v4i acc[R][C];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) acc[r][c] = v4i{0, 0, 0, 0};
        const auto step = [&](const uint8_t *stage, uint8_t *free, u32 l) {
            constexpr int n = 2 * (R + C);
            if (l + 2 * NW < lines) i8_landed<2 * n>();
            else if (l + NW < lines) i8_landed<n>();
            else i8_landed<0>();
            v4i A[2][R], B[2][C];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int r = 0; r < R; r++) A[h][r] = i8_of_line(stage + mine, lane, r, h);
#pragma unroll
                for (int c = 0; c < C; c++) B[h][c] = i8_of_line(stage + mine, lane, R + c, h);
            }
            if (l + 3 * NW < lines) src.ask(free + mine, l + 3 * NW, a.kp);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const bool in = 128 * l + 64 * h + 16 * (lane >> 4) < a.kp;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const v4i b = in ? B[h][c] : v4i{0, 0, 0, 0};
#pragma unroll
                    for (int r = 0; r < R; r++) acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[h][r], b, acc[r][c], 0, 0, 0);
                }
            }
        };
        for (u32 l = wave; l < lines;) {
            step(ring0, ring3, l);
            if ((l += NW) >= lines) break;
            step(ring1, ring0, l);
            if ((l += NW) >= lines) break;
            step(ring2, ring1, l);
            if ((l += NW) >= lines) break;
            step(ring3, ring2, l);
            l += NW;
        }
        // a thread's outputs: four rows (4 (l / 16) ..) of one column (l % 16) of tile tid / 64
        const u32 tile = wave, j = t0 + 16 * (tile % C) + (lane & 15), row = r0 + 16 * (tile / C) + 4 * (lane >> 4);
        const bool out = tile < R * C && j < run.j1 && row < a.rows;
        float scale = 0.0f, row_scale[4];
        if (out) {
            bool bad;
            const u32 col = i8_column(a, j, bad);
            if (bad) bm_raise(a.fault, a.layer, kSiteExpertId);
            scale = bad ? bm_bits_f32(0x7fc00000u) : a.qs[col];
#pragma unroll
            for (int x = 0; x < 4; x++) row_scale[x] = run.ws[min(row + x, a.rows - 1)];
        }
        i8_landed<0>();
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) *reinterpret_cast<v4i *>(ring0 + mine + (r * C + c) * 1024 + 16 * lane) = acc[r][c];
        __syncthreads();
        if (out) {
            v4i sum = v4i{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < NW; w++) sum += *reinterpret_cast<const v4i *>(ring0 + w * L::kStage + tile * 1024 + 16 * lane);
            float v[4];
#pragma unroll
            for (int x = 0; x < 4; x++) v[x] = __fmul_rn(__fmul_rn((float)sum[x], scale), row_scale[x]);
            i8_store4(a, j, row, v);
        }
        __syncthreads();
    }
}

// A few rows from their floating values: k_i8_few's product with the quantizer in front of it in every workgroup, while the first weights are on
// their way. M (a power of two, at least the rows): the waves are dealt to the rows, 4 pieces of eight values a thread at most. The codes
// go to LDS; the first workgroup leaves them and the scales in memory too.
// The values are asked for first, then three lines of weights, which stay on their way while the values become codes.
// Ahead of the two launches wherever a thread's four pieces hold the rows (us, one launch / two, bf16): 768 x 2048, one row 5.1 / 7.4, four 6.0 / 7.7, eight 6.8 /
// 7.6; 7168 x 2048, one 6.0 / 7.7, four 6.9 / 7.8, eight 7.5 / 7.9; 7168 x 7168, one 10.8 / 12.5, two 12.0 / 12.8; 8192 x 1024, eight 5.9 / 7.7. Tiles of 32 rows
// where those of 16 are more than the compute units (80 KB of LDS, one a unit): 5000 x 2048, one row 5.8 (16 rows: 8.3).
constexpr int kFewX = 8, kFewXWaves = 8; // rows at most
constexpr u32 few_x_values(u32 M) { return 64 * kFewXWaves * 8 * 4 / M; } // values a row may have
template <int ET, int M, int R>
__global__ __launch_bounds__(64 * kFewXWaves) void k_i8_few_x(I8Args a, QuantArgs qa) {
    constexpr int NW = kFewXWaves, T = 64 * NW / M, kPieces = 4; // threads a row, pieces a thread
    typedef I8Lines<2 * R> L;
    // M rows of kp. An array of its own, which no load on its way into LDS reaches: a write to it waits for none
    __shared__ __align__(16) int8_t codes[M * few_x_values(M)];
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], ring2[NW * L::kStage], ring3[NW * L::kStage];
    static_assert(R * 1024 <= L::kStage && R <= NW, "a wave's sums lie in its stage, one piece a thread");
    __shared__ u32 top[NW];
    __shared__ float scale[M];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = (u32)__builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 lines = (a.kp + 127) / 128, r0 = blockIdx.x * (16 * R), mine = wave * L::kStage;
    // the rows' values, then the first weights
    const u32 row = tid / T, first = tid % T, pieces = a.kp / 8;
    QuantPieces<ET, false, T, kPieces> in;
    in.ask(qa, min(row, qa.m - 1), first); // rows past the last are the last once more, and not multiplied
    L src;
    src.begin(lane);
#pragma unroll
    for (u32 g = 0; g < 2 * R; g++) src.from[g] = a.w + (size_t)min(r0 + 8 * g + (lane >> 3), a.rows - 1) * a.kp; // rows past the last are not stored
    // three lines whether or not there are as many (then the last once more): the wait for the values leaves a known number of loads on their way
    src.ask(ring0 + mine, min(wave, lines - 1), a.kp);
    src.ask(ring1 + mine, min(wave + NW, lines - 1), a.kp);
    src.ask(ring2 + mine, min(wave + 2 * NW, lines - 1), a.kp);
    __builtin_amdgcn_sched_barrier(0);
    i8_landed<6 * R>();
    __builtin_amdgcn_sched_barrier(0);
    float v[kPieces][8];
    bool odd = false;
    in.values(qa, min(row, qa.m - 1), first, v, odd);
    u32 most = 0;
#pragma unroll
    for (int i = 0; i < kPieces; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) most = max(most, bm_f32_bits(v[i][j]) & 0x7fffffffu);
    most = bm_max32(most);
    most = max(most, (u32)__shfl_xor((int)most, 32, 64));
    if constexpr (M < NW) {
        if (lane == 0) top[wave] = most;
        i8_meet();
        most = 0;
#pragma unroll
        for (int w = 0; w < NW / M; w++) most = max(most, top[row * (NW / M) + w]);
    }
    const I8Scale sc = i8_scale(most);
    if (first == 0) {
        scale[row] = sc.s;
        if (blockIdx.x == 0 && row < qa.m) {
            qa.scales[row] = sc.s;
            if (sc.bad) bm_raise(a.fault, a.layer, kSiteQuantColumn);
        }
    }
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const u32 c = first + i * T;
        if (c >= pieces) break;
        const uint2 word = i8_codes(v[i], sc);
        *reinterpret_cast<uint2 *>(codes + row * a.kp + 8 * c) = word;
        if (blockIdx.x == 0 && row < qa.m) *reinterpret_cast<uint2 *>(qa.codes + (size_t)row * a.kp + 8 * c) = word;
    }
    i8_meet();

    v4i acc[R];
#pragma unroll
    for (int r = 0; r < R; r++) acc[r] = v4i{0, 0, 0, 0};
    const u32 col = lane & 15;
    const auto step = [&](const uint8_t *stage, uint8_t *free, u32 l) {
        constexpr int n = 2 * R;
        if (l + 2 * NW < lines) i8_landed<2 * n>();
        else if (l + NW < lines) i8_landed<n>();
        else i8_landed<0>();
        v4i A[2][R], B[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const u32 at = 128 * l + 64 * h + 16 * (lane >> 4);
            const bool in = col < (u32)M && at < a.kp;
            const v4i b = *reinterpret_cast<const v4i *>(codes + (in ? col * a.kp + at : 0u));
            B[h] = in ? b : v4i{0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < R; r++) A[h][r] = i8_of_line(stage + mine, lane, r, h);
        }
        if (l + 3 * NW < lines) src.ask(free + mine, l + 3 * NW, a.kp);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < R; r++) acc[r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[h][r], B[h], acc[r], 0, 0, 0);
    };
    for (u32 l = wave; l < lines;) {
        step(ring0, ring3, l);
        if ((l += NW) >= lines) break;
        step(ring1, ring0, l);
        if ((l += NW) >= lines) break;
        step(ring2, ring1, l);
        if ((l += NW) >= lines) break;
        step(ring3, ring2, l);
        l += NW;
    }
    // a thread's outputs: four rows (4 (l / 16) ..) of one column (l % 16) of tile tid / 64
    const u32 out = r0 + 16 * wave + 4 * (lane >> 4);
    const bool mine_out = wave < R && col < a.m && out < a.rows;
    float row_scale[4];
    if (mine_out)
#pragma unroll
        for (int x = 0; x < 4; x++) row_scale[x] = a.ws[min(out + x, a.rows - 1)];
    i8_landed<0>();
#pragma unroll
    for (int r = 0; r < R; r++) *reinterpret_cast<v4i *>(ring0 + mine + r * 1024 + 16 * lane) = acc[r];
    __syncthreads();
    if (!mine_out) return;
    v4i sum = v4i{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; w++) sum += *reinterpret_cast<const v4i *>(ring0 + w * L::kStage + wave * 1024 + 16 * lane);
    float y[4];
#pragma unroll
    for (int x = 0; x < 4; x++) y[x] = __fmul_rn(__fmul_rn((float)sum[x], scale[col]), row_scale[x]);
    i8_store4(a, col, out, y);
}

// Many columns a matrix: BT columns x BR rows a workgroup, 128 bytes of k a step through a ring of S LDS buffers, where the loads put them
// themselves (16 bytes a lane, no register in between): while the waves multiply one step the next S - 1 are on their way, one barrier a step. A
// wave holds (BT / WT) x (BR / WR) sums in v_mfma_i32_16x16x64_i8's form.
// Large products are bound by the matrix cores and the clock that power leaves them: 4096 x 7168 x 7168 in 168 to 177 us, 2.4 to 2.5 POP/s, matrix cores busy 61 %
// of the cycles, LDS 27 %, no bank conflicts (a bare loop of these instructions on such data reaches 3.3 POP/s; the library's product of the same size takes 180 us).
// From rest the clock falls behind the first launches and comes back: of 200 in a row the first six take 173 to 180 us, the seventh to the sixtieth 185 to 225, the last
// hundred 167 to 177. Its form, 256 x 224, keeps one register of 256 in scratch memory, stored in front of the loop and fetched behind it.
// Small ones are bound by the latency of a step's loads (777 x 2000 x 1996: matrix cores 12 %), or by the way from L2 to LDS, which a smaller tile takes more often: 1024 x
// 2048 x 7168 in 64 x 64 moves 512 tiles x 56 steps x 16 KB = 470 MB in 25.2 us, 18.7 TB/s. Experts' are bound by their weights from memory.
template <int BT, int BR, int WT, int WR, int S, bool WHOLE>
struct I8Tile {
    static constexpr bool kWhole = WHOLE;
    static constexpr int kColumns = BT, kRows = BR, kRing = S, kWaves = WT * WR, kThreads = 64 * kWaves, kStage = (BT + BR) * 128;
    // a wave's loads a step, eight lines each, of columns and of rows (the last waves may repeat some of rows)
    static constexpr int RT = BT / 8 / kWaves, RR = (BR / 8 + kWaves - 1) / kWaves;
    static constexpr int TT = BT / WT / 16, TR = BR / WR / 16, H0 = (TR + 1) / 2, H1 = TR / 2; // a wave's tiles of 16, its rows in two halves
    static_assert(BT % (8 * kWaves) == 0 && BT % (16 * WT) == 0 && BR % (16 * WR) == 0 && TR > 1, "whole waves");
    static_assert(S == 2 || (S == 4 && BR % (8 * kWaves) == 0), "where steps overlap, their loads are counted: as many for every wave");
    // buffers from this one on lie past what a read's constant reaches
    static constexpr int kUp = S * kStage <= 65536 ? S : S / 2;
};

// A tile of the experts: their runs cut into tiles of BT entries, numbered through the experts in order. False: there is none of that number. The bounds
// of 256 experts are asked for at once; a run that is none has no tiles. `check`: every run is looked at, those behind the tile too, and one that
// is none raises ExpertId (one workgroup of a launch does so).
template <int BT>
__device__ __forceinline__ bool i8_find_tile(const I8Args &a, u32 tile, bool check, u32 &expert, u32 &t0) {
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

// All but the last AHEAD steps that a wave asked for have landed, and every wave is done with the buffer that is written next. (The wait as a
// builtin: the compiler counts it, where behind one in asm it would wait for the loads that follow too.)
template <class G, int AHEAD>
__device__ __forceinline__ void i8_turn() {
    constexpr int n = AHEAD * (G::RT + G::RR);
    static_assert(n < 64, "vmcnt");
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | (n >> 4) << 14); // vmcnt(n) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// Where a lane's loads begin: offsets of its lines' pieces from the tile's first column and row, and how far each goes back in the last step
// where the rows end before the piece does (to the line's first piece, which is there; the columns' are zeroed in LDS).
template <class G>
struct I8Src {
    const int8_t *q, *w; // this step's
    u32 col[G::RT], row[G::RR], back[2];
};
// The eight rows of a wave's r-th load: where there are not as many for every wave, the last ones are asked for again.
template <class G>
__device__ __forceinline__ u32 i8_row_group(u32 wave, int r) {
    const u32 group = wave * G::RR + r;
    return G::kRows % (8 * G::kWaves) == 0 ? group : min(group, (u32)G::kRows / 8 - 1);
}
template <class G>
__device__ __forceinline__ void i8_ask(I8Src<G> &s, uint8_t *buf, u32 wave, bool last) {
#pragma unroll
    for (int r = 0; r < G::RT; r++) {
        const u32 group = wave * G::RT + r;
        __builtin_amdgcn_global_load_lds((i8_gptr *)(s.q + (s.col[r] - (last ? s.back[group & 1] : 0u))), (i8_lptr *)(buf + group * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < G::RR; r++) {
        const u32 group = i8_row_group<G>(wave, r);
        __builtin_amdgcn_global_load_lds((i8_gptr *)(s.w + (s.row[r] - (last ? (group & 1 ? s.back[1] : s.back[0]) : 0u))),
                                         (i8_lptr *)(buf + G::kColumns * 128 + group * 1024), 16, 0, 0);
    }
    s.q += 128;
    s.w += 128;
}
// The columns' pieces from `have` on, in a step that has landed.
template <class G>
__device__ __forceinline__ void i8_zero_past(uint8_t *buf, u32 have) {
    for (u32 i = threadIdx.x; i < G::kColumns * 8; i += G::kThreads)
        if (((i & 7) ^ i8_swizzle(i >> 3)) >= have) *reinterpret_cast<uint4 *>(buf + 16 * i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
}

// Where a lane's reads begin, for each 64 bytes of a step: of rows and of columns. The upper buffers' carry the first one's place with them
// (and are read that far in front), so that a read's address is one register and a constant that its instruction can hold.
struct I8At {
    u32 a[2], b[2];
};
// What the matrix instructions take of 64 bytes of k of N tiles, from the FIRST on.
template <class G, int B, int N>
__device__ __forceinline__ void i8_read(v4i (&f)[N], const uint8_t *__restrict__ buf, u32 at, int first) {
    constexpr u32 up = B >= G::kUp ? (u32)G::kUp * G::kStage : 0u;
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = *reinterpret_cast<const v4i *>(buf + (int)(at - up + (first + i) * 2048));
}
template <int N, int TT>
__device__ __forceinline__ void i8_multiply(const v4i (&a)[N], const v4i (&b)[TT], v4i (*acc)[TT]) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][j], 0, 0, 0);
}
// READS of what comes next between MFMAS products of what is there.
template <int READS, int MFMAS>
__device__ __forceinline__ void i8_weave() {
#pragma unroll
    for (int i = 0; i < READS; i++) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);              // an LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, MFMAS / READS ? MFMAS / READS : 1, 0); // products
    }
}

// A step: its 128 bytes of k from buf in four parts - 64 bytes against half of the wave's rows each -, whose first part's pieces are in a0 and b0
// already; leaves the next step's there. A part's pieces are read under the products of the part before. That the two buffers are apart is
// said by restrict: else the compiler waits for the loads into one in front of every read of the other. The turn comes before the last
// part, so that the next step's reads and the loads of the one behind it go out under its products.
// FULL: more steps are left behind this one than the ring holds, so that nothing is asked of where the rows end. B: buf's number.
template <class G, int B, bool FULL>
__device__ __forceinline__ void i8_step(I8Src<G> &src, uint8_t *__restrict__ buf, uint8_t *__restrict__ next, u32 wave, u32 left, u32 tail,
                                        const I8At (&at)[2], v4i (&a0)[G::H0], v4i (&b0)[G::TT], v4i (&acc)[G::TR][G::TT]) {
    constexpr int kUp = B >= G::kUp, kNext = (B + 1) % G::kRing, kNextUp = kNext >= G::kUp;
    v4i a1[G::H1], b1[G::TT];
    i8_read<G, B>(a1, buf, at[kUp].a[0], G::H0);
    i8_multiply(a0, b0, acc);
    i8_weave<G::H1, G::H0 * G::TT>();
    i8_read<G, B>(a0, buf, at[kUp].a[1], 0);
    i8_read<G, B>(b1, buf, at[kUp].b[1], 0);
    i8_multiply(a1, b0, acc + G::H0);
    i8_weave<G::H0 + G::TT, G::H1 * G::TT>();
    i8_read<G, B>(a1, buf, at[kUp].a[1], G::H0);
    i8_multiply(a0, b1, acc);
    i8_weave<G::H1, G::H0 * G::TT>();
    if constexpr (FULL) {
        i8_turn<G, G::kRing - 2>();
        i8_ask<G>(src, buf, wave, false);
    } else if (left > 0) {
        if (G::kRing == 2 || left == 1) i8_turn<G, 0>();
        else if (left == 2) i8_turn<G, G::kRing == 2 ? 0 : 1>();
        else i8_turn<G, G::kRing - 2>();
        if (left >= (u32)G::kRing) i8_ask<G>(src, buf, wave, left == (u32)G::kRing);
        else if (left == 1 && tail < 8) i8_zero_past<G>(next, tail);
    }
    if (FULL || left > 0) {
        i8_read<G, kNext>(a0, next, at[kNextUp].a[0], 0);
        i8_read<G, kNext>(b0, next, at[kNextUp].b[0], 0);
    }
    i8_multiply(a1, b1, acc + G::H0);
    if constexpr (FULL) i8_weave<G::H0 + G::TT, G::H1 * G::TT>();
}

// The same with a whole step's pieces in registers, f for the present step and g for the next: where a part has few products, a step would be four
// waits for LDS (some 580 cycles a step of 32 x 64 sums) and is one so.
template <class G>
struct I8Whole {
    v4i a[2][G::TR], b[2][G::TT];
};
template <class G, int B>
__device__ __forceinline__ void i8_read_whole(I8Whole<G> &f, const uint8_t *__restrict__ buf, const I8At (&at)[2]) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
        i8_read<G, B>(f.a[c], buf, at[B >= G::kUp].a[c], 0);
        i8_read<G, B>(f.b[c], buf, at[B >= G::kUp].b[c], 0);
    }
}
template <class G, int B, bool FULL>
__device__ __forceinline__ void i8_step_whole(I8Src<G> &src, uint8_t *__restrict__ buf, uint8_t *__restrict__ next, u32 wave, u32 left, u32 tail,
                                              const I8At (&at)[2], const I8Whole<G> &f, I8Whole<G> &g, v4i (&acc)[G::TR][G::TT]) {
    if constexpr (FULL) {
        i8_turn<G, G::kRing - 2>();
        i8_ask<G>(src, buf, wave, false);
    } else if (left > 0) {
        if (G::kRing == 2 || left == 1) i8_turn<G, 0>();
        else if (left == 2) i8_turn<G, G::kRing == 2 ? 0 : 1>();
        else i8_turn<G, G::kRing - 2>();
        if (left >= (u32)G::kRing) i8_ask<G>(src, buf, wave, left == (u32)G::kRing);
        else if (left == 1 && tail < 8) i8_zero_past<G>(next, tail);
    }
    if (FULL || left > 0) i8_read_whole<G, (B + 1) % G::kRing>(g, next, at);
#pragma unroll
    for (int c = 0; c < 2; c++) i8_multiply(f.a[c], f.b[c], acc);
}

// Where piece p of column c lies in a line of LINE pieces: turned by the column within the pieces' largest power of two.
template <int LINE>
__device__ __forceinline__ u32 i8_turned(u32 p, u32 c) {
    constexpr u32 kPow = LINE & -LINE;
    return p ^ (c & (kPow - 1));
}

// A wave's sums as values. The matrix instruction leaves column l % 16, rows 4 (l / 16) .. + 3 of a 16 x 16 tile in lane l; the sums go through LDS
// (32 columns at a time, a wave's own part of it, four rows a piece, pieces turned by the column for the banks), so that a lane stores
// sixteen bytes of a row of y and a row's lanes are neighbours. (Straight from the registers, eight bytes a lane and 32 rows of y an
// instruction, a tile's end took 27 us; 8192 x 8192 outputs 1.2 TB/s.)
template <int ET, class G>
__device__ __forceinline__ void i8_tile_out(const I8Args &a, const I8Run &run, uint8_t *lds, u32 e0, u32 row0, const v4i (&acc)[G::TR][G::TT]) {
    constexpr int kLine = G::TR * 4, kPiecesOut = ET == kElemF32 ? 1 : 2, kValues = 4 * kPiecesOut; // a column's pieces; a lane's pieces and values a store
    constexpr int kBusy = kLine / kPiecesOut, kLanes = kBusy <= 8 ? 8 : kBusy <= 16 ? 16 : 32;        // a column's lanes: a power of two, the last ones idle
    static_assert(kLine % kPiecesOut == 0 && kBusy <= kLanes, "whole lanes");
    static_assert(G::TT % 2 == 0 && G::TT <= 4, "a lane a column, 32 at a time");
    const u32 lane = threadIdx.x & 63;
    float col_scale = 0.0f;
    if (lane < G::TT * 16 && e0 + lane < run.j1) {
        bool bad;
        const u32 col = i8_column(a, e0 + lane, bad);
        if (bad) bm_raise(a.fault, a.layer, kSiteExpertId);
        col_scale = bad ? bm_bits_f32(0x7fc00000u) : a.qs[col];
    }
    const u32 first = lane % kLanes * kPiecesOut, row = row0 + 4 * first; // this lane's pieces of every column, and its rows
    const bool mine = lane % kLanes < (u32)kBusy && row < a.rows;
    float r[kValues];
    if (mine) elem_load_some<kElemF32, kValues>(run.ws, row, a.rows - row, r);
#pragma unroll
    for (int j = 0; j < G::TT; j += 2) {
#pragma unroll
        for (int jj = 0; jj < 2; jj++) {
            const u32 t = 16 * jj + (lane & 15);
#pragma unroll
            for (int i = 0; i < G::TR; i++)
                *reinterpret_cast<v4i *>(lds + 16 * (t * kLine + i8_turned<kLine>(4 * i + (lane >> 4), t))) = acc[i][j + jj];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int n = 0; n < 32 * kLanes / 64; n++) {
            const u32 c = n * (64 / kLanes) + lane / kLanes, e = e0 + 16 * j + c;
            const float s = __shfl(col_scale, 16 * j + c, 64);
            if (!mine || e >= run.j1) continue;
            float v[kValues];
#pragma unroll
            for (int p = 0; p < kPiecesOut; p++) {
                const v4i sum = *reinterpret_cast<const v4i *>(lds + 16 * (c * kLine + i8_turned<kLine>(first + p, c)));
#pragma unroll
                for (int x = 0; x < 4; x++) v[4 * p + x] = __fmul_rn(__fmul_rn((float)sum[x], s), r[4 * p + x]);
            }
            elem_store_some<ET, kValues>(a.y, (size_t)e * a.ld + row, a.rows - row, v);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <int BT, int BR, int WT, int WR, int S, bool WHOLE, int EU>
__global__ __launch_bounds__(64 * WT * WR) __attribute__((amdgpu_waves_per_eu(EU))) void k_i8_tile(I8Args a, u32 n_row_tiles, u32 group) {
    using G = I8Tile<BT, BR, WT, WR, S, WHOLE>;
    // in this order: the larger alignment comes first
    __shared__ __align__(4096) uint8_t ring0[G::kStage];
    __shared__ __align__(2048) uint8_t ring1[G::kStage];
    __shared__ __align__(1024) uint8_t ring2[S > 2 ? G::kStage : 16];
    __shared__ __align__(512) uint8_t ring3[S > 2 ? G::kStage : 16];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = (u32)__builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the chip's eight dies in turn (b to die b % 8, each with its own L2). Neighbouring workgroups share a tile's columns across
    // the dies, and a die's workgroups four of the rows' tiles and eight of the columns'. An expert with fewer tiles of rows than dies
    // would so have its rows on every die: there (`group`) a group of its tiles of columns stays on one die, all rows of it.
    const u32 block = i8_group();
    u32 expert = 0, t0, row_tile, tile;
    if (group) {
        const u32 i = block >> 3, per = group * n_row_tiles;
        row_tile = i % per / group;
        tile = (i / per * 8 + (block & 7)) * group + i % group;
    } else {
        row_tile = block % n_row_tiles;
        tile = block / n_row_tiles;
    }
    if (!a.start) {
        t0 = tile * BT;
        if (t0 >= a.m) return;
    } else if (!i8_find_tile<BT>(a, tile, tile == 0 && row_tile == 0, expert, t0)) return;
    const u32 r0 = row_tile * BR;
    I8Run run;
    if (!i8_run(a, expert, run)) return;
    t0 = (u32)__builtin_amdgcn_readfirstlane((int)(t0 + run.j0));
    const u32 steps = (a.kp + 127) / 128, tail = (a.kp - (steps - 1) * 128) / 16; // pieces of the last step

    // columns and rows past the last are the last ones again, and not stored
    I8Src<G> src;
    src.q = a.order ? a.q : a.q + (size_t)t0 * a.kp;
    src.w = run.w + (size_t)r0 * a.kp;
    u32 col[G::RT];
#pragma unroll
    for (int r = 0; r < G::RT; r++) col[r] = min(t0 + (wave * G::RT + r) * 8 + (lane >> 3), run.j1 - 1);
    if (a.order) i8_columns<G::RT>(a, col);
#pragma unroll
    for (int r = 0; r < G::RT; r++) src.col[r] = (a.order ? col[r] : col[r] - t0) * a.kp + 16 * ((lane & 7) ^ i8_swizzle((wave * G::RT + r) * 8 + (lane >> 3)));
#pragma unroll
    for (int r = 0; r < G::RR; r++) {
        const u32 line = i8_row_group<G>(wave, r) * 8 + (lane >> 3);
        src.row[r] = (min(r0 + line, a.rows - 1) - r0) * a.kp + 16 * ((lane & 7) ^ i8_swizzle(line));
    }
#pragma unroll
    for (int r = 0; r < 2; r++) { // (a lane's piece differs between even and odd groups of eight lines only)
        const u32 piece = (lane & 7) ^ i8_swizzle(8 * r + (lane >> 3));
        src.back[r] = piece >= tail ? 16 * piece : 0;
    }

    v4i acc[G::TR][G::TT];
#pragma unroll
    for (int i = 0; i < G::TR; i++)
#pragma unroll
        for (int j = 0; j < G::TT; j++) acc[i][j] = v4i{0, 0, 0, 0};
    const u32 wt = (wave % WT) * (BT / WT), wr = BT + (wave / WT) * (BR / WR); // this wave's first lines
    I8At at[2];
#pragma unroll
    for (u32 c = 0; c < 2; c++) {
        const u32 piece = (lane & 15) * 128 + 16 * ((4 * c + (lane >> 4)) ^ i8_swizzle(lane & 15));
#pragma unroll
        for (u32 up = 0; up < 2; up++) {
            at[up].a[c] = piece + wr * 128 + up * G::kUp * G::kStage;
            at[up].b[c] = piece + wt * 128 + up * G::kUp * G::kStage;
            __asm__("" : "+v"(at[up].a[c]), "+v"(at[up].b[c])); // one register each from here on, whatever constants meet them
        }
    }
    i8_ask<G>(src, ring0, wave, steps == 1);
    if (steps > 1) i8_ask<G>(src, ring1, wave, steps == 2);
    if (S > 2 && steps > 2) i8_ask<G>(src, ring2, wave, steps == 3);
    if (S > 2 && steps > 3) i8_ask<G>(src, ring3, wave, steps == 4);
    if (steps >= (u32)S) i8_turn<G, S - 1>();
    else i8_turn<G, 0>();
    if (steps == 1 && tail < 8) i8_zero_past<G>(ring0, tail);
    u32 left = steps - 1;
    if constexpr (WHOLE) {
        // (rings of an even number of buffers: the two sets of registers change places with every step)
        I8Whole<G> f, g;
        i8_read_whole<G, 0>(f, ring0, at);
        if constexpr (S == 2) {
            for (; left >= 4; left -= 2) {
                i8_step_whole<G, 0, true>(src, ring0, ring1, wave, 0, 0, at, f, g, acc);
                i8_step_whole<G, 1, true>(src, ring1, ring0, wave, 0, 0, at, g, f, acc);
            }
            for (;;) {
                i8_step_whole<G, 0, false>(src, ring0, ring1, wave, left, tail, at, f, g, acc);
                if (left-- == 0) break;
                i8_step_whole<G, 1, false>(src, ring1, ring0, wave, left, tail, at, g, f, acc);
                if (left-- == 0) break;
            }
        } else {
            for (; left >= 8; left -= 4) {
                i8_step_whole<G, 0, true>(src, ring0, ring1, wave, 0, 0, at, f, g, acc);
                i8_step_whole<G, 1, true>(src, ring1, ring2, wave, 0, 0, at, g, f, acc);
                i8_step_whole<G, 2, true>(src, ring2, ring3, wave, 0, 0, at, f, g, acc);
                i8_step_whole<G, 3, true>(src, ring3, ring0, wave, 0, 0, at, g, f, acc);
            }
            for (;;) {
                i8_step_whole<G, 0, false>(src, ring0, ring1, wave, left, tail, at, f, g, acc);
                if (left-- == 0) break;
                i8_step_whole<G, 1, false>(src, ring1, ring2, wave, left, tail, at, g, f, acc);
                if (left-- == 0) break;
                i8_step_whole<G, 2, false>(src, ring2, ring3, wave, left, tail, at, f, g, acc);
                if (left-- == 0) break;
                i8_step_whole<G, 3, false>(src, ring3, ring0, wave, left, tail, at, g, f, acc);
                if (left-- == 0) break;
            }
        }
    } else {
        static_assert(WHOLE || S == 2, "parts of a step in a ring of two");
        v4i a0[G::H0], b0[G::TT];
        i8_read<G, 0>(a0, ring0, at[0].a[0], 0);
        i8_read<G, 0>(b0, ring0, at[0].b[0], 0);
        for (; left >= 4; left -= 2) {
            i8_step<G, 0, true>(src, ring0, ring1, wave, 0, 0, at, a0, b0, acc);
            i8_step<G, 1, true>(src, ring1, ring0, wave, 0, 0, at, a0, b0, acc);
        }
        for (;;) {
            i8_step<G, 0, false>(src, ring0, ring1, wave, left, tail, at, a0, b0, acc);
            if (left-- == 0) break;
            i8_step<G, 1, false>(src, ring1, ring0, wave, left, tail, at, a0, b0, acc);
            if (left-- == 0) break;
        }
    }
    __syncthreads(); // the buffers are the sums' from here
    constexpr u32 kPart = G::TR * 2048, kEven = G::kStage / kPart; // a wave's part, and how many lie in the first buffer
    static_assert(G::kWaves <= 2 * kEven, "every part lies in one buffer");
    uint8_t *part = wave < kEven ? ring0 + wave * kPart : ring1 + (wave - kEven) * kPart;
    if (a.et == kElemF32) i8_tile_out<kElemF32, G>(a, run, part, t0 + wt, r0 + (wr - BT), acc);
    else if (a.et == kElemF16) i8_tile_out<kElemF16, G>(a, run, part, t0 + wt, r0 + (wr - BT), acc);
    else i8_tile_out<kElemBF16, G>(a, run, part, t0 + wt, r0 + (wr - BT), acc);
}

template <int BT, int BR, int WT, int WR, int S, bool WHOLE, int EU>
static hipError_t tile_launch(const Launch &L, const I8Args &a, u32 entries) {
    const u32 row_tiles = (a.rows + BR - 1) / BR;
    u32 tiles = (entries + BT - 1) / BT;
    if (a.start) tiles = entries / BT + (a.n_experts < entries ? a.n_experts : entries); // at most a ragged tile an expert
    const u32 group = a.start && row_tiles < 8 ? 2 : 0;
    if (group) tiles = (tiles + 8 * group - 1) / (8 * group) * (8 * group);
    hipLaunchKernelGGL((k_i8_tile<BT, BR, WT, WR, S, WHOLE, EU>), i8_grid((uint64_t)tiles * row_tiles, 64 * WT * WR), dim3(64 * WT * WR), 0, L.stream, a, row_tiles, group);
    return hipGetLastError();
}

template <int R, int C, int NW>
static hipError_t few_launch(const Launch &L, const I8Args &a, u32 entries) {
    const u32 z = a.start ? 1u : (entries + 16 * C - 1) / (16 * C);
    hipLaunchKernelGGL((k_i8_few<R, C, NW>), dim3((a.rows + 16 * R - 1) / (16 * R), a.start ? a.n_experts : 1u, z < 65535u ? z : 65535u), dim3(64 * NW), 0,
                       L.stream, a);
    return hipGetLastError();
}

template <int ET, int M, int R>
static void few_x_launch(const Launch &L, const I8Args &a, const QuantArgs &q) {
    hipLaunchKernelGGL((k_i8_few_x<ET, M, R>), dim3((a.rows + 16 * R - 1) / (16 * R)), dim3(64 * kFewXWaves), 0, L.stream, a, q);
}
template <int ET, int M>
static void few_x_by_rows(const Launch &L, const I8Args &a, const QuantArgs &q) {
    if ((a.rows + 15) / 16 > 256) few_x_launch<ET, M, 2>(L, a, q);
    else few_x_launch<ET, M, 1>(L, a, q);
}
template <int ET>
static void few_x_by_columns(const Launch &L, const I8Args &a, const QuantArgs &q) {
    if (a.m == 1) few_x_by_rows<ET, 1>(L, a, q);
    else if (a.m == 2) few_x_by_rows<ET, 2>(L, a, q);
    else if (a.m <= 4) few_x_by_rows<ET, 4>(L, a, q);
    else few_x_by_rows<ET, 8>(L, a, q);
}

hipError_t i8_gemm_x(const Launch &L, const int8_t *w, const float *ws, int rows, int k, const void *x, int x_et, int64_t ld_x, int m, int8_t *codes,
                     float *scales, void *y, int et, int64_t ld) {
    const u32 kp = (u32)i8_row_bytes(k), M = m <= 1 ? 1 : m <= 2 ? 2 : m <= 4 ? 4 : 8;
    if (m <= kFewX && k >= 8 && kp <= few_x_values(M)) {
        const I8Args a = {w, ws, (u32)rows, kp, codes, scales, (u32)m, nullptr, nullptr, 0, 0, (u32)m, 1, y, (size_t)ld, et, L.fault, L.layer};
        const QuantArgs q = {x, nullptr, (size_t)ld_x, (u32)m, (u32)k, kp, nullptr, codes, scales, L.rule, L.fault, L.layer};
        if (x_et == kElemF32) few_x_by_columns<kElemF32>(L, a, q);
        else if (x_et == kElemF16) few_x_by_columns<kElemF16>(L, a, q);
        else few_x_by_columns<kElemBF16>(L, a, q);
        return hipGetLastError();
    }
    const hipError_t e = i8_quantize(L, x, nullptr, x_et, ld_x, m, k, nullptr, codes, scales);
    return e != hipSuccess ? e : i8_gemm(L, w, ws, 1, rows, k, codes, scales, m, nullptr, nullptr, 0, 0, y, et, ld);
}

// The forms, by what a workgroup has: columns x rows, its waves and its LDS buffers.
enum I8Form : u32 {
    kFew16x16,      // k_i8_few: 16 x 16, waves sharing k
    kFew16x32,      // 16 x 32
    kFew16x32Three, // the same by three waves
    kFew32x32,
    kTile32x64Ring4, // k_i8_tile, steps in a ring of four or two
    kTile32x64,
    kTile64x64Ring4,
    kTile64x64,
    kTile64x128,
    kTile64x256,
    kTile128x128,
    kTile256x224,
    kTile256x256,
};

// Which form: all give the same bits. us on MI355X, bf16 out, weights of three sets in turn, the chosen form's first.
//   One matrix. Large tiles are the better the more of them there are, and whole rounds of 256 compute units count: a round of 256 x 256 tiles takes
//   64 units of time, of 256 x 224 57, of two 128 x 128 a unit 39. (4096 x 7168 x 7168: 512 tiles of 224 rows are two rounds, 179, 448 of 256 take
//   the same two, 198, 128 x 128 223; 4096 cubed 58, 90, 66; 8192 cubed 453, 507, 538; 4096 x 2048 x 7168, the 128 x 128 first, 59, 80, 69.)
//   Below some hundred large tiles the smaller ones fill the card. 64 x 64 with four steps in flight while they are one round of two a unit: 1024 x 2048 x 7168 25.2
//   (64 x 128: 36.1, 128 x 128: 37.8), 256 x 7168 x 2048 10.0 (12.9, 14.5); with two steps, five a unit, up to three: 1280 x 2048 x 2048 12.8 (64 x 128: 14.8), 1536 rows 12.7 (14.2), but
//   2048 16.8 (15.6). Then 64 x 128 for little more than a round of two, 700 x 7168 x 2048 18.5 (128 x 128: 19.5), and 128 x 128: 1024 x 7168 x 2048 21.0 (64 x 128: 27.3). 32 x 64
//   while they are one round: 256 x 2048 x 7168 13.2 (64 x 64: 14.3); two rounds lose, 1280 x 512 x 4096 13.1 (11.0). Short rows need no four steps: 640 x 1024 x 512 in 64 x 64 with two
//   steps 4.4 (four: 4.8), 400 x 1500 x 1024 5.9 (6.5).
//   Where tiles of at most 32 x 32 are no more than the compute units, a workgroup's waves share a row's k (k_i8_few), in the smallest tile that is one
//   round: 34 x 544 x 8064 in 16 x 16 5.6 (16 x 32: 7.0, 32 x 64 whole rows 13), 64 x 2048 x 7168 in 16 x 32 6.5 (32 x 32: 7.9; 12.8), 128 x 2048 x 7168 in 32 x 32 8.1 (16 x 32:
//   11.2; 12.9), 24 x 7168 x 2048 5.1 (7.1), one row of 2048 x 7168 4.9, of 7168 x 7168 9.6; two rounds lose, 64 x 7168 x 2048 8.2 (32 x 64: 7.5).
//   Experts, by slots an expert. From 352 on 256 x 256: 375 slots, 64 experts, 1024 x 2048 88.9 (128 x 128: 94.9), 1024 slots, 32 experts, 7168 x 2048 589 (638, 64 x
//   256: 699); from 144 on 128 x 128: 250 slots, 64 experts, 1024 x 2048 70.9 (256 x 256: 75.8, 64 x 256: 80.4), 150 slots, 7168 x 2048 295 (341, 317), 256 slots, 128 experts, 768 x 2048
//   102 (113, 115); then 64 x 256: 128 slots, 768 x 2048 73.1 (128 x 128: 77.5, 64 x 128: 79), 2048 x 768 85 (89, 89); 32 slots 45.2 (64 x 128: 52), one round of tiles; more of them in 64 x 128: 64
//   slots 59.5 (64 x 256: 63.5), 42 slots, 64 experts, 7168 x 2048 190.5 (193); 8 slots an expert in 32 x 64 37.5 (64 x 256: 39.8), one slot 20 (24; waves sharing k 25); one token's
//   eight slots by waves sharing k 6.6 (32 x 64: 9.1).
//   While 64 x 64 tiles are few, so that a compute unit has one to four: short runs in 32 x 64 with four steps in flight, 20 tokens, top 4 of 52, 288 x 6224 13.9 (two steps 24.5, 64 x
//   64 25.7), 152 tokens, top 5 of 54, 688 x 3376 35.5 (64 x 256: 48.4), 100 tokens, top 2 of 16, 1024 x 4096 15.8 (18.3, 27.4); longer ones in 64 x 64, with four steps up to one a
//   unit, 100 tokens, top 8 of 16, 768 x 2048 10.7 (two steps 12.4, 64 x 256 17.4), with two steps behind that, 400 tokens, top 2 of 8, 2048 x 2048 13.6 (four 16.1, 64 x 256 17.8), 600
//   tokens, 1000 x 1000 9.7 (10.1, 13.8); least of all by waves sharing k, 40 tokens, top 4 of 32, 96 x 4000 7.0 (32 x 64: 10.2).
//   A die's group of two tiles of columns (k_i8_tile) in these: 128 slots, 768 x 2048 72, without 88 (its weights are then fetched 1.8 times: 369 MB at 5.5 TB/s); 256 slots 102, without
//   117. Where a run's rows are eight tiles or more it loses (64 experts, 7168 x 2048 190.8 without, 201 with); dies with whole ranges of the experts lose there too (202) and gain
//   little here (69).
//   Experts' gathered columns past 4 GiB, which the tiles' 32-bit offsets do not reach, go by waves sharing k however many there are: 599187 tokens of 7168, top 4 of 256, 2048
//   rows 409 ms, one token fewer, in 256 x 256, 33 to 38. One token's experts launch every expert's tiles, most with nothing to do: top 8 of 256, 2048 x 7168 31 with the
//   quantizer, 7168 x 2048 45 (57344 workgroups, 1792 of them with work), of 128, 768 x 2048 9.9.
// n_experts 0: one matrix, n its columns; else n slots. reach: the tiles' offsets of gathered columns, 32 bits, hold the columns.
static I8Form i8_form(u32 n_experts, u32 rows, u32 kp, u32 n, bool reach) {
    const auto up = [](u32 x, u32 y) { return (x + y - 1) / y; };
    const auto tiles = [&](u32 bt, u32 br) { return (uint64_t)up(n, bt) * up(rows, br); };
    if (n_experts) {
        if (n <= 32 || !reach) return kFew16x32Three;
        const u32 each = n / n_experts, runs = n < n_experts ? n : n_experts;
        // 64 x 64 tiles: every run has one, and half a one more than its slots fill
        const uint64_t small = (uint64_t)std::max(runs, n / 64 + runs / 2) * up(rows, 64);
        if (each <= 16 && small <= 64) return kFew32x32;
        if (each < 24 && small <= 600) return kTile32x64Ring4;
        if (each >= 24 && small <= 256) return kTile64x64Ring4;
        if (each >= 24 && small <= 1024) return kTile64x64;
        if (each >= 352) return kTile256x256;
        if (each >= 144) return kTile128x128;
        // 64 x 256 where its tiles (half a tile more an expert) are one round of two a compute unit, or the runs long
        if (each >= 96 || (each >= 12 && (uint64_t)(n / 64 + n_experts / 2) * up(rows, 256) <= 512)) return kTile64x256;
        return each >= 12 ? kTile64x128 : kTile32x64;
    }
    if (tiles(16, 16) <= 256) return kFew16x16;
    if (tiles(16, 32) <= 256) return kFew16x32;
    if (n <= 16) return kFew16x32Three;
    if (n <= 32 || tiles(32, 32) <= 256) return kFew32x32;
    if (tiles(32, 64) <= 256) return kTile32x64Ring4;
    if (tiles(64, 64) <= 512 && kp > 1024) return kTile64x64Ring4;
    if (tiles(64, 64) <= 768) return kTile64x64;
    if (tiles(256, 256) >= 96) {
        const uint64_t by256 = 64 * ((tiles(256, 256) + 255) / 256), by224 = 57 * ((tiles(256, 224) + 255) / 256), by128 = 39 * ((tiles(128, 128) + 511) / 512);
        if (by256 <= by224 && by256 <= by128) return kTile256x256;
        return by224 <= by128 ? kTile256x224 : kTile128x128;
    }
    return tiles(64, 128) <= 640 ? kTile64x128 : kTile128x128;
}
static bool i8_reach(bool gathered, int n_cols, u32 kp) { return !gathered || (uint64_t)n_cols * kp <= 0xffffffffu; }

int i8_gemm_form(int n_experts, int rows, int k, int n_cols, int n_slots, int top_k) {
    static const struct {
        u32 columns, rows, waves, buffers;
    } of[] = {{16, 16, 8, 4}, {16, 32, 4, 4}, {16, 32, 3, 4}, {32, 32, 4, 4}, {32, 64, 2, 4}, {32, 64, 2, 2}, {64, 64, 4, 4},
              {64, 64, 4, 2}, {64, 128, 4, 2}, {64, 256, 4, 2}, {128, 128, 4, 2}, {256, 224, 8, 2}, {256, 256, 8, 2}};
    const u32 kp = (u32)i8_row_bytes(k);
    const auto &f = of[i8_form((u32)n_experts, (u32)rows, kp, (u32)(n_experts ? n_slots : n_cols), i8_reach(n_experts && top_k > 0, n_cols, kp))];
    return (int)(f.columns | f.rows << 10 | f.waves << 20 | f.buffers << 24);
}

hipError_t i8_gemm(const Launch &L, const int8_t *w, const float *ws, int n_experts, int rows, int k, const int8_t *q, const float *qs, int n_cols,
                   const uint32_t *order, const uint32_t *start, int n_slots, int top_k, void *y, int et, int64_t ld) {
    const I8Args a = {w, ws, (u32)rows, (u32)i8_row_bytes(k), q, qs, (u32)n_cols, order, start, (u32)n_slots, (u32)top_k, (u32)n_cols, (u32)n_experts,
                      y, (size_t)ld, et, L.fault, L.layer};
    const u32 n = start ? (u32)n_slots : (u32)n_cols;
    switch (i8_form(start ? a.n_experts : 0, a.rows, a.kp, n, i8_reach(order != nullptr, n_cols, a.kp))) {
    case kFew16x16: return few_launch<1, 1, 8>(L, a, n);
    case kFew16x32: return few_launch<2, 1, 4>(L, a, n);
    case kFew16x32Three: return few_launch<2, 1, 3>(L, a, n);
    case kFew32x32: return few_launch<2, 2, 4>(L, a, n);
    case kTile32x64Ring4: return tile_launch<32, 64, 1, 2, 4, true, 2>(L, a, n);
    case kTile32x64: return tile_launch<32, 64, 1, 2, 2, true, 2>(L, a, n);
    case kTile64x64Ring4: return tile_launch<64, 64, 2, 2, 4, true, 2>(L, a, n);
    case kTile64x64: return tile_launch<64, 64, 2, 2, 2, true, 2>(L, a, n);
    case kTile64x128: return tile_launch<64, 128, 1, 4, 2, true, 2>(L, a, n);
    case kTile64x256: return tile_launch<64, 256, 1, 4, 2, true, 2>(L, a, n);
    case kTile128x128: return tile_launch<128, 128, 2, 2, 2, true, 2>(L, a, n);
    case kTile256x224: return tile_launch<256, 224, 4, 2, 2, false, 2>(L, a, n);
    case kTile256x256: return tile_launch<256, 256, 4, 2, 2, false, 2>(L, a, n);
    }
    return hipErrorInvalidValue;
}

} // namespace bmk
