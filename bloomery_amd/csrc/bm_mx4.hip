// Experts in microscaled 4-bit floating point: rows in blocks of 32 values, four bits each and a power of two a block. The quantizer and its way back, products of
// such rows with such columns (one matrix, or experts' matrices over the runs that a router made), and the experts' whole step for a few
// tokens whose values stay in floating point.
//
//   code   one sign, two exponent and one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6; two to a byte, the even value's in the low half
//   scale  2^(b - 127), b a byte; 255 is NaN
//   block  b = clamp(exponent of max |x| - 2, 0, 254) in biased exponents, a code the nearest value to x / 2^(b - 127), halves to the even code,
//          held to 6: the division is by a power of two, so a code depends on nothing but x
//   value  y = sum over blocks of 2^(bt + bw - 254) times the sum of 32 products, in f32
//
// A row of codes is 16 bytes a block, a row of scales one, rounded up to 16.
#include "bm_lines.hpp"

#include <algorithm>
#include <type_traits>

namespace bmk {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------------------------------------------ quantizer

struct Mx4Rows {
    const void *x, *u; // u: the second input of a gate rule
    size_t ld;
    u32 m, k, kp, ks; // bytes of a row's codes and scales
    const u32 *live;  // rows at or past it stay as they are (NULL: all m)
    uint8_t *codes, *scales;
    GateRule rule;
    u32 *fault, layer;
};

template <int CTRL>
__device__ __forceinline__ u32 quad_swap(u32 v) {
    return (u32)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// Four lanes' largest.
__device__ __forceinline__ u32 quad_max(u32 v) {
    v = max(v, quad_swap<0xb1>(v));
    return max(v, quad_swap<0x4e>(v));
}

// Eight values of a block that four neighbouring lanes hold: their codes, and the block's scale. The largest magnitude's biased exponent less 2 is the scale's
// byte; the conversion takes that byte as an exponent's bits, 0 for 2^-127, divides exactly, rounds to the nearest code, halves to even, and holds to 6.
__device__ __forceinline__ u32 mx4_block(const float (&v)[8], u32 &scale) {
    u32 most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = max(most, bm_f32_bits(v[j]) & 0x7fffffffu);
    most = quad_max(most) >> 23;
    const bool bad = most == 255;
    scale = bad ? 255 : most > 2 ? most - 2 : 0;
    const float s = bm_bits_f32(scale << 23);
    u32 word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], s, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], s, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], s, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], s, 3);
    return bad ? 0u : word;
}

// A wave takes sixteen blocks of a row, sixteen bytes of its scales: a lane eight values, four lanes a block, whose maximum is two exchanges between
// neighbours, so that nothing goes through LDS and a value is read once. Memory bounds it: 4096 x 7168 bf16 17 us, 4.3 TB/s of 74 MB; 16 x 2048 f32 2.4 us, a launch. Behind the gate rule
// the vector units do, by the rule's exponential and its exact division: 4096 x 7168 bf16 38 us, 3.5 TB/s (f32 47 us, 5.3 TB/s), 2664 x 2048 f16 10.3, 666 x 2048 5.1.
template <int ET, bool GLU>
__global__ __launch_bounds__(256) void k_mx4_quantize(Mx4Rows a) {
    const u32 lane = threadIdx.x & 63, units = a.ks / 16, unit = group_index() * 4 + (threadIdx.x >> 6), row = unit / units;
    const u32 m = a.live ? min(a.m, *a.live) : a.m;
    if (row >= m) return;
    const u32 block = unit % units * 16 + (lane >> 2), c = block * 32 + 8 * (lane & 3), have = c < a.k ? a.k - c : 0;
    float v[8];
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.0f;
    if (have) {
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
    if (GLU && odd) bm_raise(a.fault, a.layer, kSiteF32Product);
    u32 scale;
    const u32 word = mx4_block(v, scale);
    if ((lane & 3) == 0) {
        a.scales[(size_t)row * a.ks + block] = (uint8_t)scale;
        if (scale == 255) bm_raise(a.fault, a.layer, kSiteQuantColumn);
    }
    if (16 * block < a.kp) *reinterpret_cast<u32 *>(a.codes + (size_t)row * a.kp + c / 2) = word;
}

// Eight codes as values.
__device__ __forceinline__ void mx4_values(u32 word, u32 scale, float (&v)[8]) {
    const float s = bm_bits_f32(scale << 23);
    const v2f p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 1),
              p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 3);
    v[0] = p0[0], v[1] = p0[1], v[2] = p1[0], v[3] = p1[1], v[4] = p2[0], v[5] = p2[1], v[6] = p3[0], v[7] = p3[1];
}

// And back, the same shares: 4096 x 7168 to bf16 12.3 us, 6.0 TB/s (the codes come from the last-level cache).
template <int ET>
__global__ __launch_bounds__(256) void k_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, u32 m, u32 k, u32 kp, u32 ks, void *y, size_t ld) {
    const u32 lane = threadIdx.x & 63, units = ks / 16, unit = group_index() * 4 + (threadIdx.x >> 6), row = unit / units;
    const u32 block = unit % units * 16 + (lane >> 2), c = block * 32 + 8 * (lane & 3);
    if (row >= m || c >= k) return;
    float v[8];
    mx4_values(*reinterpret_cast<const u32 *>(codes + (size_t)row * kp + c / 2), scales[(size_t)row * ks + block], v);
    elem_store_some<ET, 8>(y, (size_t)row * ld + c, k - c, v);
}

hipError_t mx4_quantize(const Launch &L, const void *x, const void *u, int et, int64_t ld, int m, int k, const uint32_t *live, uint8_t *codes,
                        uint8_t *scales) {
    const Mx4Rows a = {x, u, (size_t)ld, (u32)m, (u32)k, (u32)mx4_row_bytes(k), (u32)mx4_row_scales(k), live, codes, scales, L.rule, L.fault, L.layer};
    const dim3 grid = group_grid(((uint64_t)m * (a.ks / 16) + 3) / 4, 256);
    if (u) {
        if (et == kElemF32) hipLaunchKernelGGL((k_mx4_quantize<kElemF32, true>), grid, dim3(256), 0, L.stream, a);
        else if (et == kElemF16) hipLaunchKernelGGL((k_mx4_quantize<kElemF16, true>), grid, dim3(256), 0, L.stream, a);
        else hipLaunchKernelGGL((k_mx4_quantize<kElemBF16, true>), grid, dim3(256), 0, L.stream, a);
    } else {
        if (et == kElemF32) hipLaunchKernelGGL((k_mx4_quantize<kElemF32, false>), grid, dim3(256), 0, L.stream, a);
        else if (et == kElemF16) hipLaunchKernelGGL((k_mx4_quantize<kElemF16, false>), grid, dim3(256), 0, L.stream, a);
        else hipLaunchKernelGGL((k_mx4_quantize<kElemBF16, false>), grid, dim3(256), 0, L.stream, a);
    }
    return hipGetLastError();
}

hipError_t mx4_dequantize(const Launch &L, const uint8_t *codes, const uint8_t *scales, int m, int k, void *y, int et, int64_t ld) {
    const u32 kp = (u32)mx4_row_bytes(k), ks = (u32)mx4_row_scales(k);
    const dim3 grid = group_grid(((uint64_t)m * (ks / 16) + 3) / 4, 256);
    if (et == kElemF32) hipLaunchKernelGGL((k_mx4_dequantize<kElemF32>), grid, dim3(256), 0, L.stream, codes, scales, (u32)m, (u32)k, kp, ks, y, (size_t)ld);
    else if (et == kElemF16) hipLaunchKernelGGL((k_mx4_dequantize<kElemF16>), grid, dim3(256), 0, L.stream, codes, scales, (u32)m, (u32)k, kp, ks, y, (size_t)ld);
    else hipLaunchKernelGGL((k_mx4_dequantize<kElemBF16>), grid, dim3(256), 0, L.stream, codes, scales, (u32)m, (u32)k, kp, ks, y, (size_t)ld);
    return hipGetLastError();
}

// -------------------------------------------------------------------------------------------------- product

struct Mx4Args {
    const uint8_t *w, *ws; // rows (of one matrix, or of an expert's) x kp, x ks
    u32 rows, kp, ks;
    const uint8_t *q, *qs; // columns
    u32 m;                 // columns of one matrix's product
    const u32 *order;      // experts: entry j's slot (NULL: entry j reads column j)
    const u32 *start;      // experts' runs (NULL: one matrix)
    u32 n_slots, top_k, n_cols, n_experts;
    void *y;
    size_t ld;
    int et;
    u32 *fault, layer;
};

// A run of entries and the matrix they meet.
struct Mx4Run {
    u32 j0, j1;
    const uint8_t *w, *ws;
};
__device__ __forceinline__ bool mx4_run(const Mx4Args &a, u32 e, Mx4Run &r) {
    if (!a.start) {
        r = Mx4Run{0, a.m, a.w, a.ws};
        return true;
    }
    const u32 j0 = a.start[e], j1 = a.start[e + 1];
    if (j0 > j1 || j1 > a.n_slots) { // no run of a table over these slots
        if (threadIdx.x == 0) bm_raise(a.fault, a.layer, kSiteExpertId);
        return false;
    }
    r = Mx4Run{j0, j1, a.w + (size_t)e * a.rows * a.kp, a.ws + (size_t)e * a.rows * a.ks};
    return j1 > j0;
}

// Sixteen rows by sixteen columns, 128 values of k: lane l holds a block of row (column) l % 16, four blocks in turn, and its scale in byte H of
// a word; it gets column l % 16, rows 4 (l / 16) .. + 3. Of a 128-byte line, eight blocks, lane l takes blocks 2 (l / 16) and the next, one for each of two
// instructions: their scales are two neighbouring bytes.
template <int H>
__device__ __forceinline__ v4f mx4_mfma(v4i w, v4i q, v4f acc, u32 ws, u32 qs) {
    const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {q[0], q[1], q[2], q[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, H, (int)ws, H, (int)qs);
}
// Two scales, 1 in the place of those from block `blocks` on, whose codes are zeros.
__device__ __forceinline__ u32 mx4_scales(u32 two, u32 block, u32 blocks) {
    return block + 1 < blocks ? two : block < blocks ? (two & 0xffu) | 0x7f00u : 0x7f7fu;
}
__device__ __forceinline__ u32 mx4_two(const uint8_t *p) { return *reinterpret_cast<const uint16_t *>(p); }
// What the matrix instructions take of line group t (sixteen lines) of a stage: piece 2 (l / 16) + h of the lines.
__device__ __forceinline__ v4i mx4_of_line(const uint8_t *stage, u32 lane, int t, int h) {
    return *reinterpret_cast<const v4i *>(stage + t * 2048 + (lane & 15) * 128 + 16 * ((2 * (lane >> 4) + h) ^ line_swizzle(lane & 15)));
}

// The sums of a tile's waves, in the waves' order, are a thread's outputs: four rows (4 (l / 16) ..) of one column.
template <int NW, class L>
__device__ __forceinline__ v4f mx4_join(const uint8_t *ring, u32 tile, u32 lane) {
    v4f sum = *reinterpret_cast<const v4f *>(ring + tile * 1024 + 16 * lane);
#pragma unroll
    for (int w = 1; w < NW; w++) sum += *reinterpret_cast<const v4f *>(ring + w * L::kStage + tile * 1024 + 16 * lane);
    return sum;
}

// Few columns a matrix: 16 R rows a workgroup against 16 C columns, its NW waves dealing the row's lines among them, each through a ring of four
// stages of its own, two on their way while one is multiplied and the fourth is asked for; a line's scales come straight to registers, asked for with it. The
// waves' sums meet in LDS. Few workgroups have a row's whole k to get through, so the way from memory bounds it, and with k over the waves a workgroup has as
// many lines on their way as it has waves and stages: 24 x 7168 x 2048 4.9 us (with whole rows of k in tiles of 32 x 64 5.8), one row of 7168 x 7168 7.7, 3.5 TB/s.
template <int R, int C, int NW>
__global__ __launch_bounds__(64 * NW) void k_mx4_few(Mx4Args a) {
    typedef Lines<2 * (R + C)> L;
    constexpr int kLoads = 3 * (R + C); // of a stage: 2 (R + C) of lines, R + C of scales
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], ring2[NW * L::kStage], ring3[NW * L::kStage];
    static_assert(R * C * 1024 <= L::kStage && R * C <= NW, "a wave's sums lie in its stage, one piece a thread");
    const u32 lane = threadIdx.x & 63, wave = (u32)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Mx4Run run;
    if (!mx4_run(a, blockIdx.y, run)) return;
    const u32 r0 = blockIdx.x * (16 * R), lines = (a.kp + 127) / 128, mine = wave * L::kStage, blocks = a.kp / 16, at = 2 * (lane >> 4);
    L src;
    src.begin(lane);
    const uint8_t *scales[R + C];
#pragma unroll
    for (u32 g = 0; g < 2 * R; g++) src.from[g] = (const int8_t *)run.w + (size_t)min(r0 + 8 * g + (lane >> 3), a.rows - 1) * a.kp; // rows past the last are not stored
#pragma unroll
    for (u32 r = 0; r < R; r++) scales[r] = run.ws + (size_t)min(r0 + 16 * r + (lane & 15), a.rows - 1) * a.ks + at;
    for (u32 t0 = run.j0 + blockIdx.z * (16 * C); t0 < run.j1; t0 += gridDim.z * (16 * C)) {
        u32 col[3 * C];
#pragma unroll
        for (u32 g = 0; g < 2 * C; g++) col[g] = min(t0 + 8 * g + (lane >> 3), run.j1 - 1);
#pragma unroll
        for (u32 c = 0; c < C; c++) col[2 * C + c] = min(t0 + 16 * c + (lane & 15), run.j1 - 1);
        if (a.order) run_columns(a, col);
#pragma unroll
        for (u32 g = 0; g < 2 * C; g++) src.from[2 * R + g] = (const int8_t *)a.q + (size_t)col[g] * a.kp;
#pragma unroll
        for (u32 c = 0; c < C; c++) scales[R + c] = a.qs + (size_t)col[2 * C + c] * a.ks + at;
        u32 s0[R + C], s1[R + C], s2[R + C], s3[R + C];
        const auto ask = [&](uint8_t *stage, u32 (&s)[R + C], u32 l) {
#pragma unroll
            for (int i = 0; i < R + C; i++) s[i] = mx4_two(scales[i] + 8 * l);
            __builtin_amdgcn_sched_barrier(0);
            src.ask(stage + mine, l, a.kp);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (wave < lines) ask(ring0, s0, wave);
        if (wave + NW < lines) ask(ring1, s1, wave + NW);
        if (wave + 2 * NW < lines) ask(ring2, s2, wave + 2 * NW);
        v4f acc[R][C];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) acc[r][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        const auto step = [&](const uint8_t *stage, u32 (&s)[R + C], uint8_t *free, u32 (&next)[R + C], u32 l) {
            if (l + 2 * NW < lines) loads_landed<2 * kLoads>();
            else if (l + NW < lines) loads_landed<kLoads>();
            else loads_landed<0>();
            v4i A[2][R], B[2][C];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int r = 0; r < R; r++) A[h][r] = mx4_of_line(stage + mine, lane, r, h);
#pragma unroll
                for (int c = 0; c < C; c++) B[h][c] = mx4_of_line(stage + mine, lane, R + c, h);
            }
            u32 two[R + C];
#pragma unroll
            for (int i = 0; i < R + C; i++) two[i] = mx4_scales(s[i], 8 * l + at, blocks);
            if (l + 3 * NW < lines) ask(free, next, l + 3 * NW);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const bool in = 8 * l + at + h < blocks;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const v4i b = in ? B[h][c] : v4i{0, 0, 0, 0};
#pragma unroll
                    for (int r = 0; r < R; r++) acc[r][c] = h ? mx4_mfma<1>(A[h][r], b, acc[r][c], two[r], two[R + c]) : mx4_mfma<0>(A[h][r], b, acc[r][c], two[r], two[R + c]);
                }
            }
        };
        for (u32 l = wave; l < lines;) {
            step(ring0, s0, ring3, s3, l);
            if ((l += NW) >= lines) break;
            step(ring1, s1, ring0, s0, l);
            if ((l += NW) >= lines) break;
            step(ring2, s2, ring1, s1, l);
            if ((l += NW) >= lines) break;
            step(ring3, s3, ring2, s2, l);
            l += NW;
        }
        const u32 tile = wave, j = t0 + 16 * (tile % C) + (lane & 15), row = r0 + 16 * (tile / C) + 4 * (lane >> 4);
        const bool out = tile < R * C && j < run.j1 && row < a.rows;
        bool bad = false;
        if (out) {
            run_column(a, j, bad);
            if (bad) bm_raise(a.fault, a.layer, kSiteExpertId);
        }
        loads_landed<0>();
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) *reinterpret_cast<v4f *>(ring0 + mine + (r * C + c) * 1024 + 16 * lane) = acc[r][c];
        __syncthreads();
        if (out) {
            const v4f sum = mx4_join<NW, L>(ring0, tile, lane);
            float v[4];
#pragma unroll
            for (int x = 0; x < 4; x++) v[x] = bad ? bm_bits_f32(0x7fc00000u) : sum[x];
            run_store4(a, j, row, v);
        }
        __syncthreads();
    }
}

// A few rows from their floating values: k_mx4_few's product with the quantizer in front of it in every workgroup, while the first weights are on
// their way. M (a power of two, at least the rows): the waves are dealt to the rows, PC pieces of eight values a thread at most, four threads a
// block. Codes and scales go to LDS; the first workgroup leaves them in memory too. One launch for two, whose cost it is: 1 x 768 x 2048 f32 3.9 us,
// as much as k_mx4_few alone. What it costs more is every workgroup's reading of all rows: bf16, us,
// 16 x 1024 against 4096 and 8192 rows of weights 4.3, 5.2 (two launches 7.2, 7.5), 16 x 2048 6.0, 6.8 (8.4), 32 x 1024 6.0, 6.8 (8.5), 1 x 32768 18.9, 33.5 (19.8, 38.3), f32 16 x 2048 6.5, 7.7 (8.4);
// but twice the values in two turns 8.9, 9.7 (24 x 2048, two launches 8.0), and more than 8192 rows of weights, several rounds of workgroups, 8 x 2048 against 16000 9.7 (8.2).
constexpr int kMx4FewX = 32, kMx4FewXWaves = 8; // rows at most
constexpr u32 mx4_few_x_values(u32 M, u32 PC) { return 64 * kMx4FewXWaves * 8 * PC / M; } // values a row may have
template <int ET, int M, int R, int PC>
__global__ __launch_bounds__(64 * kMx4FewXWaves) void k_mx4_few_x(Mx4Args a, Mx4Rows qa) {
    constexpr int NW = kMx4FewXWaves, T = 64 * NW / M, V = kElemPiece<ET>, P = 8 / V, C = M <= 16 ? 1 : 2;    // threads a row, loads a piece, columns' tiles
    constexpr u32 kRow = mx4_few_x_values(M, PC) / 2 + 16, kRowScales = mx4_few_x_values(M, PC) / 32; // a row's bytes in LDS, sixteen more for the banks
    typedef Lines<2 * R> L;
    constexpr int kLoads = 3 * R;
    __shared__ __align__(16) uint8_t codes[M * kRow], marks[M * kRowScales];
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], ring2[NW * L::kStage], ring3[NW * L::kStage];
    static_assert(R * C * 1024 <= L::kStage && R * C <= NW, "a wave's sums lie in its stage, one piece a thread");
    const u32 tid = threadIdx.x, lane = tid & 63, wave = (u32)__builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 lines = (a.kp + 127) / 128, r0 = blockIdx.x * (16 * R), mine = wave * L::kStage, blocks = a.kp / 16, at = 2 * (lane >> 4);
    // the rows' values, then the first weights
    const u32 row = tid / T, first = tid % T, pieces = a.kp / 4, whole = qa.k / 8;
    const size_t from = (size_t)min(row, qa.m - 1) * qa.ld; // rows past the last are the last once more, and not multiplied
    uint4 x[PC][P];
#pragma unroll
    for (int i = 0; i < PC; i++)
#pragma unroll
        for (int p = 0; p < P; p++) x[i][p] = elem_piece<ET>(qa.x, from + 8 * min(first + i * T, whole - 1) + p * V);
    L src;
    src.begin(lane);
    const uint8_t *scales[R];
#pragma unroll
    for (u32 g = 0; g < 2 * R; g++) src.from[g] = (const int8_t *)a.w + (size_t)min(r0 + 8 * g + (lane >> 3), a.rows - 1) * a.kp; // rows past the last are not stored
#pragma unroll
    for (u32 r = 0; r < R; r++) scales[r] = a.ws + (size_t)min(r0 + 16 * r + (lane & 15), a.rows - 1) * a.ks + at;
    u32 s0[R], s1[R], s2[R], s3[R];
    const auto ask = [&](uint8_t *stage, u32 (&s)[R], u32 l) {
#pragma unroll
        for (int i = 0; i < R; i++) s[i] = mx4_two(scales[i] + 8 * l);
        __builtin_amdgcn_sched_barrier(0);
        src.ask(stage + mine, l, a.kp);
        __builtin_amdgcn_sched_barrier(0);
    };
    // three lines whether or not there are as many (then the last once more): the wait for the values leaves a known number of loads on their way
    ask(ring0, s0, min(wave, lines - 1));
    ask(ring1, s1, min(wave + NW, lines - 1));
    ask(ring2, s2, min(wave + 2 * NW, lines - 1));
    loads_landed<3 * kLoads>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < PC; i++) {
        const u32 c = first + i * T;
        if (c >= pieces) break; // (a block's four threads together)
        float v[8];
#pragma unroll
        for (int p = 0; p < P; p++) {
            float e[V];
            elem_unpack<ET>(x[i][p], e);
#pragma unroll
            for (int j = 0; j < V; j++) v[p * V + j] = c < whole ? e[j] : 0.0f;
        }
        if (c == whole && (qa.k & 7)) elem_load_some<ET, 8>(qa.x, from + 8 * c, qa.k - 8 * c, v);
        u32 scale;
        const u32 word = mx4_block(v, scale);
        const bool mark = (c & 3) == 0, leave = blockIdx.x == 0 && row < qa.m;
        *reinterpret_cast<u32 *>(codes + row * kRow + 4 * c) = word;
        if (mark) marks[row * kRowScales + c / 4] = (uint8_t)scale;
        if (leave) *reinterpret_cast<u32 *>(qa.codes + (size_t)row * a.kp + 4 * c) = word;
        if (leave && mark) {
            qa.scales[(size_t)row * a.ks + c / 4] = (uint8_t)scale;
            if (scale == 255) bm_raise(qa.fault, qa.layer, kSiteQuantColumn);
        }
    }
    if (blockIdx.x == 0 && row < qa.m)
        for (u32 b = blocks + first; b < a.ks; b += T) qa.scales[(size_t)row * a.ks + b] = 0;
    lds_meet();

    v4f acc[R][C];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) acc[r][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const u32 col = lane & 15;
    const auto step = [&](const uint8_t *stage, u32 (&s)[R], uint8_t *free, u32 (&next)[R], u32 l) {
        if (l + 2 * NW < lines) loads_landed<2 * kLoads>();
        else if (l + NW < lines) loads_landed<kLoads>();
        else loads_landed<0>();
        v4i A[2][R], B[2][C];
        u32 two[R], q[C];
        const u32 block = 8 * l + at;
        const bool here = M >= 16 || col < (u32)M;
#pragma unroll
        for (int c = 0; c < C; c++) {
            q[c] = 0x7f7fu;
            if (here && block < blocks) q[c] = mx4_scales(mx4_two(marks + (16 * c + col) * kRowScales + block), block, blocks);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool in = here && block + h < blocks;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const v4i b = *reinterpret_cast<const v4i *>(codes + (in ? (16 * c + col) * kRow + 16 * (block + h) : 0u));
                B[h][c] = in ? b : v4i{0, 0, 0, 0};
            }
#pragma unroll
            for (int r = 0; r < R; r++) A[h][r] = mx4_of_line(stage + mine, lane, r, h);
        }
#pragma unroll
        for (int r = 0; r < R; r++) two[r] = mx4_scales(s[r], block, blocks);
        if (l + 3 * NW < lines) ask(free, next, l + 3 * NW);
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) acc[r][c] = mx4_mfma<0>(A[0][r], B[0][c], acc[r][c], two[r], q[c]);
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) acc[r][c] = mx4_mfma<1>(A[1][r], B[1][c], acc[r][c], two[r], q[c]);
    };
    for (u32 l = wave; l < lines;) {
        step(ring0, s0, ring3, s3, l);
        if ((l += NW) >= lines) break;
        step(ring1, s1, ring0, s0, l);
        if ((l += NW) >= lines) break;
        step(ring2, s2, ring1, s1, l);
        if ((l += NW) >= lines) break;
        step(ring3, s3, ring2, s2, l);
        l += NW;
    }
    const u32 out = r0 + 16 * (wave / C) + 4 * (lane >> 4), j = 16 * (wave % C) + col;
    loads_landed<0>();
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) *reinterpret_cast<v4f *>(ring0 + mine + (r * C + c) * 1024 + 16 * lane) = acc[r][c];
    __syncthreads();
    if (wave >= R * C || j >= a.m || out >= a.rows) return;
    const v4f sum = mx4_join<NW, L>(ring0, wave, lane);
    const float y[4] = {sum[0], sum[1], sum[2], sum[3]};
    run_store4(a, j, out, y);
}

// Many columns a matrix: BT columns x BR rows a workgroup, 128 bytes of k a step through two LDS buffers, where the loads put them themselves (16 bytes a
// lane, no register in between), and 32 bytes of scales a column and a row, four steps' worth, through two more: while the waves multiply one step
// the next is on its way, one barrier a step. A wave holds (BT / WT) x (BR / WR) sums in v_mfma_scale_f32_16x16x128_f8f6f4's form; Q of its tiles of rows are a part
// of a step (0: all).
// What bounds it: in large products the way into LDS, some 32 bytes a cycle and unit, so that an instruction of 16 cycles wants tiles of 256 x 256 (8192 cubed 247 us,
// 4.5 PFLOP/s, of 6.5 that the instructions alone reach on random codes; 256 x 128 302, 128 x 128 328), whose 128 sums a lane leave no registers for a
// third set: scales come four steps at once, offsets go into the buffers' descriptors, and no step has a branch (without these 203 registers
// and more went to scratch). In small ones the way from memory: 777 x 2000 x 1996 8 us at 1.6 tiles a unit.
template <int BT, int BR, int WT, int WR, int Q>
struct Mx4Tile {
    static constexpr int kColumns = BT, kRows = BR, kLines = BT + BR, kWaves = WT * WR, kThreads = 64 * kWaves, kStage = kLines * 128, kMarks = kLines * 32;
    // a wave's loads: eight lines each, of columns and of rows, and 32 lines' scales every four steps (the last waves may repeat some)
    static constexpr int RT = BT / 8 / kWaves, RR = (BR / 8 + kWaves - 1) / kWaves, RG = (kLines / 32 + kWaves - 1) / kWaves;
    static constexpr int TT = BT / WT / 16, TR = BR / WR / 16, kPart = Q ? Q : TR; // a wave's tiles of 16
    static_assert(BT % (8 * kWaves) == 0 && BT % (16 * WT) == 0 && BR % (16 * WR) == 0 && BT % 32 == 0 && BR % 32 == 0 && TR % kPart == 0, "whole waves and parts");
    // buffers from this one on lie past what a read's constant reaches
    static constexpr int kUp = 2 * kStage <= 65536 ? 2 : 1;
};

// What a wave asked for has landed, and every wave is done with the buffer that is written next.
__device__ __forceinline__ void mx4_turn() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// Where a tile's loads begin: its columns and rows and their scales as buffers that end where the matrices do - what lies past their ends comes as zeros,
// so that a line may run on behind its row's end -, and a lane's offsets in them.
template <class G>
struct Mx4Src {
    const uint8_t *q, *w, *qs, *ws;
    u32 q_end, w_end, qs_end, ws_end; // bytes
    u32 at, mark_at;                  // this step's place in the lines, this group's in the scales
    u32 col[G::RT], row[G::RR], mark[G::RG];
};
__device__ __forceinline__ u32 mx4_end(size_t bytes) { return bytes < 0xffffffffu ? (u32)bytes : 0xffffffffu; }
__device__ __forceinline__ void mx4_load(const uint8_t *from, u32 end, uint8_t *to, u32 lane_at, u32 at) {
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(from), 0, (int)end, 0x00027000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_to *)to, 16, (int)lane_at, (int)at, 0, 0);
}
template <class G>
__device__ __forceinline__ u32 mx4_mark_group(u32 wave, int r) {
    const u32 group = wave * G::RG + r;
    return (G::kLines / 32) % G::kWaves == 0 ? group : min(group, (u32)G::kLines / 32 - 1);
}
template <class G>
__device__ __forceinline__ void mx4_ask(Mx4Src<G> &s, uint8_t *buf, u32 wave) {
#pragma unroll
    for (int r = 0; r < G::RT; r++) mx4_load(s.q, s.q_end, buf + (wave * G::RT + r) * 1024, s.col[r], s.at);
#pragma unroll
    for (int r = 0; r < G::RR; r++) mx4_load(s.w, s.w_end, buf + G::kColumns * 128 + tile_row_group<G>(wave, r) * 1024, s.row[r], s.at);
    s.at += 128;
}
// Four steps' scales, 32 bytes a line, two pieces, which change places in every second eight lines: a step's of sixteen lines come from all the banks.
__device__ __forceinline__ u32 mx4_mark_turn(u32 line) { return 2 * (line & 8); }
template <class G>
__device__ __forceinline__ void mx4_ask_marks(Mx4Src<G> &s, uint8_t *marks, u32 wave) {
#pragma unroll
    for (int r = 0; r < G::RG; r++) {
        const u32 group = mx4_mark_group<G>(wave, r);
        const bool columns = group < G::kColumns / 32;
        mx4_load(columns ? s.qs : s.ws, columns ? s.qs_end : s.ws_end, marks + group * 1024, s.mark[r], s.mark_at);
    }
    s.mark_at += 32;
}
// In a step that has landed, the columns' blocks from `have` on become zeros, and the scales there 1, the rows' too.
template <class G>
__device__ __forceinline__ void mx4_zero_past(uint8_t *buf, uint8_t *marks, u32 place, u32 have) {
    for (u32 i = threadIdx.x; i < G::kColumns * 8; i += G::kThreads)
        if (((i & 7) ^ line_swizzle(i >> 3)) >= have) *reinterpret_cast<uint4 *>(buf + 16 * i) = make_uint4(0, 0, 0, 0);
    for (u32 i = threadIdx.x; i < G::kLines; i += G::kThreads)
        for (u32 b = have; b < 8; b++) marks[32 * i + (place ^ mx4_mark_turn(i)) + b] = 127;
    __syncthreads();
}

// Where a lane's reads begin: the lines' (TileAt, by buffer) and the scales'.
struct Mx4At {
    TileAt line[2];
    u32 sa, sb, turn;
};
// A step's scales: two blocks' of each of a wave's tiles.
template <class G>
struct Mx4Marks {
    u32 a[G::TR], b[G::TT];
    __device__ __forceinline__ void read(const uint8_t *__restrict__ marks, u32 place, const Mx4At &at) {
        const uint8_t *mine = marks + (place ^ at.turn);
#pragma unroll
        for (int j = 0; j < G::TT; j++) b[j] = mx4_two(mine + at.sb + j * 512);
#pragma unroll
        for (int i = 0; i < G::TR; i++) a[i] = mx4_two(mine + at.sa + i * 512);
    }
};
// Where a step's scales lie: four steps' in one half, the next four's in the other; and their place in a line's.
template <class G>
__device__ __forceinline__ u32 mx4_mark_half(u32 step) { return (step >> 2 & 1) * G::kMarks; }
__device__ __forceinline__ u32 mx4_mark_place(u32 step) { return (step & 3) * 8; }
template <int H, int N, int TT>
__device__ __forceinline__ void mx4_multiply(const v4i (&a)[N], const v4i (&b)[TT], const u32 *sa, const u32 (&sb)[TT], v4f (*acc)[TT]) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = mx4_mfma<H>(a[i], b[j], acc[i][j], sa[i], sb[j]);
}

// What a step does beside its products: between kFull, where the one behind the next is asked for, kNext, where there is none behind the next, which
// is the last, and kLast, with none behind it. No branch stands in a step but in kNext: the compiler would carry the products past it.
enum Mx4Steps { kFull, kNext, kLast };
struct Mx4Way {
    u32 step, tail, wave; // this step's number, and the blocks of the last one
};
template <class G, Mx4Steps STEP, class F>
__device__ __forceinline__ void mx4_next(Mx4Src<G> &src, uint8_t *buf, uint8_t *next, uint8_t *marks, const Mx4Way &way, F read) {
    if constexpr (STEP == kLast) return;
    mx4_turn();
    uint8_t *half = marks + mx4_mark_half<G>(way.step + 1);
    const u32 place = mx4_mark_place(way.step + 1);
    if (STEP == kNext && way.tail < 8) mx4_zero_past<G>(next, half, place, way.tail);
    read(half, place);
    if (STEP == kNext) return;
    mx4_ask<G>(src, buf, way.wave);
}

// A step in parts: Q of a wave's tiles of rows against 64 bytes of k each. The first part's pieces and the scales are in registers already, and
// the next step's are left there. A part's pieces are read under the products of the part before. That the two buffers are apart is said by
// restrict: else the compiler waits for the loads into one in front of every read of the other. The turn comes before the last part, so
// that the next step's reads and the loads of the one behind it go out under its products. B: the buffer's number.
template <class G>
struct Mx4Parts {
    v4i a[G::kPart], b[G::TT];
    Mx4Marks<G> s;
    template <int B>
    __device__ __forceinline__ void begin(const uint8_t *buf, const uint8_t *marks, const Mx4At &at) {
        constexpr int up = B >= G::kUp;
        s.read(marks, 0, at);
        tile_read<G, B>(a, buf, at.line[up].a[0], 0);
        tile_read<G, B>(b, buf, at.line[up].b[0], 0);
    }
    template <int B, Mx4Steps STEP>
    __device__ __forceinline__ void step(Mx4Src<G> &src, uint8_t *__restrict__ buf, uint8_t *__restrict__ next, uint8_t *__restrict__ marks, Mx4Way &way,
                                         const Mx4At &at, v4f (&acc)[G::TR][G::TT]) {
        constexpr int Q = G::kPart, N = G::TR / Q, up = B >= G::kUp, nextUp = 1 - B >= G::kUp;
        v4i part[2][Q], b1[G::TT];
#pragma unroll
        for (int i = 0; i < Q; i++) part[0][i] = a[i];
#pragma unroll
        for (int p = 0; p < 2 * N - 1; p++) {
            tile_read<G, B>(part[(p + 1) & 1], buf, at.line[up].a[(p + 1) / N], (p + 1) % N * Q); // the next part's
            if (p == N - 1) tile_read<G, B>(b1, buf, at.line[up].b[1], 0);
            if (p < N) mx4_multiply<0>(part[p & 1], b, s.a + p % N * Q, s.b, acc + p % N * Q);
            else mx4_multiply<1>(part[p & 1], b1, s.a + p % N * Q, s.b, acc + p % N * Q);
            if (p == N - 1) tile_weave<Q + G::TT, Q * G::TT>();
            else tile_weave<Q, Q * G::TT>();
        }
        const Mx4Marks<G> mine = s;
        mx4_next<G, STEP>(src, buf, next, marks, way, [&](const uint8_t *m, u32 place) {
            s.read(m, place, at);
            tile_read<G, 1 - B>(a, next, at.line[nextUp].a[0], 0);
            tile_read<G, 1 - B>(b, next, at.line[nextUp].b[0], 0);
        });
        mx4_multiply<1>(part[1], b1, mine.a + (N - 1) * Q, mine.b, acc + (N - 1) * Q);
        if constexpr (STEP == kFull) tile_weave<Q + 2 * G::TT + G::TR, Q * G::TT>();
        way.step++;
    }
};

// The same with a whole step's pieces in registers, two sets that change places with every step: where a part has few products, a step would be many
// waits for LDS and is one so.
template <class G>
struct Mx4Whole {
    struct Set {
        v4i a[2][G::TR], b[2][G::TT];
        Mx4Marks<G> s;
    } set[2];
    template <int B>
    __device__ __forceinline__ void read(const uint8_t *__restrict__ buf, const uint8_t *__restrict__ marks, u32 place, const Mx4At &at) {
        constexpr int up = B >= G::kUp;
        set[B].s.read(marks, place, at);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            tile_read<G, B>(set[B].a[c], buf, at.line[up].a[c], 0);
            tile_read<G, B>(set[B].b[c], buf, at.line[up].b[c], 0);
        }
    }
    template <int B>
    __device__ __forceinline__ void begin(const uint8_t *buf, const uint8_t *marks, const Mx4At &at) { read<B>(buf, marks, 0, at); }
    template <int B, Mx4Steps STEP>
    __device__ __forceinline__ void step(Mx4Src<G> &src, uint8_t *__restrict__ buf, uint8_t *__restrict__ next, uint8_t *__restrict__ marks, Mx4Way &way,
                                         const Mx4At &at, v4f (&acc)[G::TR][G::TT]) {
        mx4_next<G, STEP>(src, buf, next, marks, way, [&](const uint8_t *m, u32 place) { read<1 - B>(next, m, place, at); });
        mx4_multiply<0>(set[B].a[0], set[B].b[0], set[B].s.a, set[B].s.b, acc);
        mx4_multiply<1>(set[B].a[1], set[B].b[1], set[B].s.a, set[B].s.b, acc);
        way.step++;
    }
};

// A wave's sums as values. The matrix instruction leaves column l % 16, rows 4 (l / 16) .. + 3 of a 16 x 16 tile in lane l; the sums go through LDS
// (32 columns at a time, a wave's own part of it, four rows a piece, pieces turned by the column for the banks), so that a lane stores
// sixteen bytes of a row of y and a row's lanes are neighbours.
template <int ET, class G>
__device__ __forceinline__ void mx4_tile_out(const Mx4Args &a, const Mx4Run &run, uint8_t *lds, u32 e0, u32 row0, const v4f (&acc)[G::TR][G::TT]) {
    constexpr int kLine = G::TR * 4, kPiecesOut = ET == kElemF32 ? 1 : 2, kValues = 4 * kPiecesOut; // a column's pieces; a lane's pieces and values a store
    constexpr int kBusy = kLine / kPiecesOut, kLanes = kBusy <= 8 ? 8 : kBusy <= 16 ? 16 : 32;        // a column's lanes: a power of two, the last ones idle
    static_assert(kLine % kPiecesOut == 0 && kBusy <= kLanes, "whole lanes");
    static_assert(G::TT % 2 == 0 && G::TT <= 4, "a lane a column, 32 at a time");
    const u32 lane = threadIdx.x & 63;
    bool bad = false;
    if (a.order && lane < G::TT * 16 && e0 + lane < run.j1) {
        run_column(a, e0 + lane, bad);
        if (bad) bm_raise(a.fault, a.layer, kSiteExpertId);
    }
    const unsigned long long none = __ballot(bad);
    const u32 first = lane % kLanes * kPiecesOut, row = row0 + 4 * first; // this lane's pieces of every column, and its rows
    const bool mine = lane % kLanes < (u32)kBusy && row < a.rows;
#pragma unroll
    for (int j = 0; j < G::TT; j += 2) {
#pragma unroll
        for (int jj = 0; jj < 2; jj++) {
            const u32 t = 16 * jj + (lane & 15);
#pragma unroll
            for (int i = 0; i < G::TR; i++)
                *reinterpret_cast<v4f *>(lds + 16 * (t * kLine + tile_turned<kLine>(4 * i + (lane >> 4), t))) = acc[i][j + jj];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int n = 0; n < 32 * kLanes / 64; n++) {
            const u32 c = n * (64 / kLanes) + lane / kLanes, e = e0 + 16 * j + c;
            if (!mine || e >= run.j1) continue;
            float v[kValues];
#pragma unroll
            for (int p = 0; p < kPiecesOut; p++) {
                const v4f sum = *reinterpret_cast<const v4f *>(lds + 16 * (c * kLine + tile_turned<kLine>(first + p, c)));
#pragma unroll
                for (int x = 0; x < 4; x++) v[4 * p + x] = none >> (16 * j + c) & 1 ? bm_bits_f32(0x7fc00000u) : sum[x];
            }
            elem_store_some<ET, kValues>(a.y, (size_t)e * a.ld + row, a.rows - row, v);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <int BT, int BR, int WT, int WR, int Q, int EU>
__global__ __launch_bounds__(64 * WT * WR) __attribute__((amdgpu_waves_per_eu(EU))) void k_mx4_tile(Mx4Args a, u32 n_row_tiles, u32 group) {
    using G = Mx4Tile<BT, BR, WT, WR, Q>;
    // in this order: the larger alignment comes first
    __shared__ __align__(4096) uint8_t ring0[G::kStage];
    __shared__ __align__(2048) uint8_t ring1[G::kStage];
    __shared__ __align__(1024) uint8_t marks[2 * G::kMarks];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = (u32)__builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the chip's eight dies in turn (b to die b % 8, each with its own L2). Neighbouring workgroups share a tile's columns across
    // the dies, and a die's workgroups four of the rows' tiles and eight of the columns'. An expert with fewer tiles of rows than dies
    // would so have its rows on every die: there (`group`) a group of its tiles of columns stays on one die, all rows of it.
    const u32 block = group_index();
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
    } else if (!run_tile<BT>(a, tile, tile == 0 && row_tile == 0, expert, t0)) return;
    const u32 r0 = row_tile * BR;
    Mx4Run run;
    if (!mx4_run(a, expert, run)) return;
    t0 = (u32)__builtin_amdgcn_readfirstlane((int)(t0 + run.j0));
    const u32 steps = (a.kp + 127) / 128, last = steps - 1;

    // columns and rows past the last are the last ones again, and not stored
    Mx4Src<G> src;
    {
        const size_t c0 = a.order ? 0 : t0, columns = (a.start ? a.n_cols : a.m) - c0, rows = a.rows - r0;
        src.q = a.q + c0 * a.kp, src.q_end = mx4_end(columns * a.kp);
        src.qs = a.qs + c0 * a.ks, src.qs_end = mx4_end(columns * a.ks);
        src.w = run.w + (size_t)r0 * a.kp, src.w_end = mx4_end(rows * a.kp);
        src.ws = run.ws + (size_t)r0 * a.ks, src.ws_end = mx4_end(rows * a.ks);
    }
    src.at = src.mark_at = 0;
    u32 col[G::RT + G::RG];
#pragma unroll
    for (int r = 0; r < G::RT; r++) col[r] = min(t0 + (wave * G::RT + r) * 8 + (lane >> 3), run.j1 - 1);
#pragma unroll
    for (int r = 0; r < G::RG; r++) col[G::RT + r] = min(t0 + mx4_mark_group<G>(wave, r) * 32 + (lane >> 1), run.j1 - 1); // (of a group of rows: not used)
    if (a.order) run_columns(a, col);
    else
#pragma unroll
        for (int r = 0; r < G::RT + G::RG; r++) col[r] -= t0;
#pragma unroll
    for (int r = 0; r < G::RT; r++) src.col[r] = col[r] * a.kp + 16 * ((lane & 7) ^ line_swizzle((wave * G::RT + r) * 8 + (lane >> 3)));
#pragma unroll
    for (int r = 0; r < G::RR; r++) {
        const u32 line = tile_row_group<G>(wave, r) * 8 + (lane >> 3);
        src.row[r] = (min(r0 + line, a.rows - 1) - r0) * a.kp + 16 * ((lane & 7) ^ line_swizzle(line));
    }
#pragma unroll
    for (int r = 0; r < G::RG; r++) {
        const u32 line = mx4_mark_group<G>(wave, r) * 32 + (lane >> 1);
        const u32 row = min(r0 + line - (u32)BT, a.rows - 1) - r0;
        src.mark[r] = (line < (u32)BT ? col[G::RT + r] : row) * a.ks + (16 * (lane & 1) ^ mx4_mark_turn(line));
    }

    v4f acc[G::TR][G::TT];
#pragma unroll
    for (int i = 0; i < G::TR; i++)
#pragma unroll
        for (int j = 0; j < G::TT; j++) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const u32 wt = (wave % WT) * (BT / WT), wr = BT + (wave / WT) * (BR / WR); // this wave's first lines
    Mx4At at;
    at.sa = (wr + (lane & 15)) * 32 + 2 * (lane >> 4);
    at.sb = (wt + (lane & 15)) * 32 + 2 * (lane >> 4);
    at.turn = mx4_mark_turn(lane);
#pragma unroll
    for (u32 c = 0; c < 2; c++) {
        const u32 piece = (lane & 15) * 128 + 16 * ((2 * (lane >> 4) + c) ^ line_swizzle(lane & 15));
#pragma unroll
        for (u32 up = 0; up < 2; up++) {
            at.line[up].a[c] = piece + wr * 128 + up * G::kUp * G::kStage;
            at.line[up].b[c] = piece + wt * 128 + up * G::kUp * G::kStage;
            __asm__("" : "+v"(at.line[up].a[c]), "+v"(at.line[up].b[c])); // one register each from here on, whatever constants meet them
        }
    }
    Mx4Way way = {0, a.kp / 16 - 8 * last, wave};
    typename std::conditional<Q == 0, Mx4Whole<G>, Mx4Parts<G>>::type f;
    mx4_ask_marks<G>(src, marks, wave);
    if (last & 1) { // an even number of steps: the first and the last two by themselves, pairs between them
        mx4_ask<G>(src, ring0, wave);
        mx4_turn();
        mx4_ask<G>(src, ring1, wave);
        f.template begin<0>(ring0, marks, at);
    } else {
        mx4_ask<G>(src, ring1, wave);
        mx4_turn();
        if (last == 0 && way.tail < 8) mx4_zero_past<G>(ring1, marks, 0, way.tail);
        if (last) mx4_ask<G>(src, ring0, wave);
        f.template begin<1>(ring1, marks, at);
        if (last) {
            mx4_ask_marks<G>(src, marks + G::kMarks, wave);
            f.template step<1, kFull>(src, ring1, ring0, marks, way, at, acc);
        }
    }
    if (last) {
        while (way.step + 1 < last) {
            // in the first pair of four steps, or the second and third of them, the next four's scales; those of steps 4 to 7 may be on their way
            if ((way.step & 3) < 2 && way.step != 1) mx4_ask_marks<G>(src, marks + (~way.step >> 2 & 1) * G::kMarks, wave);
            f.template step<0, kFull>(src, ring0, ring1, marks, way, at, acc);
            f.template step<1, kFull>(src, ring1, ring0, marks, way, at, acc);
        }
        f.template step<0, kNext>(src, ring0, ring1, marks, way, at, acc);
    }
    f.template step<1, kLast>(src, ring1, ring0, marks, way, at, acc);
    __syncthreads(); // the buffers are the sums' from here
    constexpr u32 kPart = G::TR * 2048, kEven = G::kStage / kPart; // a wave's part, and how many lie in the first buffer
    static_assert(G::kWaves <= 2 * kEven, "every part lies in one buffer");
    uint8_t *part = wave < kEven ? ring0 + wave * kPart : ring1 + (wave - kEven) * kPart;
    if (a.et == kElemF32) mx4_tile_out<kElemF32, G>(a, run, part, t0 + wt, r0 + (wr - BT), acc);
    else if (a.et == kElemF16) mx4_tile_out<kElemF16, G>(a, run, part, t0 + wt, r0 + (wr - BT), acc);
    else mx4_tile_out<kElemBF16, G>(a, run, part, t0 + wt, r0 + (wr - BT), acc);
}

template <int BT, int BR, int WT, int WR, int Q, int EU>
static hipError_t mx4_tile_launch(const Launch &L, const Mx4Args &a, u32 entries) {
    const u32 row_tiles = (a.rows + BR - 1) / BR;
    u32 tiles = (entries + BT - 1) / BT;
    if (a.start) tiles = entries / BT + (a.n_experts < entries ? a.n_experts : entries); // at most a ragged tile an expert
    const u32 group = a.start && row_tiles < 8 ? 2 : 0;
    if (group) tiles = (tiles + 8 * group - 1) / (8 * group) * (8 * group);
    hipLaunchKernelGGL((k_mx4_tile<BT, BR, WT, WR, Q, EU>), group_grid((uint64_t)tiles * row_tiles, 64 * WT * WR), dim3(64 * WT * WR), 0, L.stream, a, row_tiles, group);
    return hipGetLastError();
}

template <int R, int C, int NW>
static hipError_t mx4_few_launch(const Launch &L, const Mx4Args &a, u32 entries) {
    const u32 z = a.start ? 1u : (entries + 16 * C - 1) / (16 * C);
    hipLaunchKernelGGL((k_mx4_few<R, C, NW>), dim3((a.rows + 16 * R - 1) / (16 * R), a.start ? a.n_experts : 1u, z < 65535u ? z : 65535u), dim3(64 * NW), 0,
                       L.stream, a);
    return hipGetLastError();
}

template <int ET, int M, int R, int PC>
static void mx4_few_x_launch(const Launch &L, const Mx4Args &a, const Mx4Rows &q) {
    hipLaunchKernelGGL((k_mx4_few_x<ET, M, R, PC>), dim3((a.rows + 16 * R - 1) / (16 * R)), dim3(64 * kMx4FewXWaves), 0, L.stream, a, q);
}
template <int ET, int M>
static void mx4_few_x_by_rows(const Launch &L, const Mx4Args &a, const Mx4Rows &q) {
    const bool two = (a.rows + 15) / 16 > 256;
    if (2 * a.kp <= mx4_few_x_values(M, 4)) {
        if (two) mx4_few_x_launch<ET, M, 2, 4>(L, a, q);
        else mx4_few_x_launch<ET, M, 1, 4>(L, a, q);
    } else if (two) mx4_few_x_launch<ET, M, 2, 8>(L, a, q);
    else mx4_few_x_launch<ET, M, 1, 8>(L, a, q);
}
template <int ET>
static void mx4_few_x_by_columns(const Launch &L, const Mx4Args &a, const Mx4Rows &q) {
    if (a.m == 1) mx4_few_x_by_rows<ET, 1>(L, a, q);
    else if (a.m == 2) mx4_few_x_by_rows<ET, 2>(L, a, q);
    else if (a.m <= 4) mx4_few_x_by_rows<ET, 4>(L, a, q);
    else if (a.m <= 8) mx4_few_x_by_rows<ET, 8>(L, a, q);
    else if (a.m <= 16) mx4_few_x_by_rows<ET, 16>(L, a, q);
    else mx4_few_x_by_rows<ET, 32>(L, a, q);
}

hipError_t mx4_gemm_x(const Launch &L, const uint8_t *w, const uint8_t *ws, int rows, int k, const void *x, int x_et, int64_t ld_x, int m, uint8_t *codes,
                      uint8_t *scales, void *y, int et, int64_t ld) {
    const u32 kp = (u32)mx4_row_bytes(k), ks = (u32)mx4_row_scales(k), M = m <= 1 ? 1 : m <= 2 ? 2 : m <= 4 ? 4 : m <= 8 ? 8 : m <= 16 ? 16 : 32;
    if (m <= kMx4FewX && k >= 8 && 2 * kp <= mx4_few_x_values(M, 8) && rows <= 256 * 32) {
        const Mx4Args a = {w, ws, (u32)rows, kp, ks, codes, scales, (u32)m, nullptr, nullptr, 0, 0, (u32)m, 1, y, (size_t)ld, et, L.fault, L.layer};
        const Mx4Rows q = {x, nullptr, (size_t)ld_x, (u32)m, (u32)k, kp, ks, nullptr, codes, scales, L.rule, L.fault, L.layer};
        if (x_et == kElemF32) mx4_few_x_by_columns<kElemF32>(L, a, q);
        else if (x_et == kElemF16) mx4_few_x_by_columns<kElemF16>(L, a, q);
        else mx4_few_x_by_columns<kElemBF16>(L, a, q);
        return hipGetLastError();
    }
    const hipError_t e = mx4_quantize(L, x, nullptr, x_et, ld_x, m, k, nullptr, codes, scales);
    return e != hipSuccess ? e : mx4_gemm(L, w, ws, 1, rows, k, codes, scales, m, nullptr, nullptr, 0, 0, y, et, ld);
}

// The forms, by what a workgroup has: columns x rows, its waves and its LDS buffers.
enum Mx4Form : u32 {
    kMx4Few16x16, // k_mx4_few: waves sharing k
    kMx4Few16x32,
    kMx4Few32x32,
    kMx4Tile32x64, // k_mx4_tile
    kMx4Tile64x64,
    kMx4Tile128x128,
    kMx4Tile256x128,
    kMx4Tile256x256,
};

// Which form, us on MI355X, bf16 out, weights of three sets in turn (two for experts), the chosen form's first.
//   One matrix. While tiles of at most 32 x 32 are no more than the compute units a workgroup's waves share a row's k, in the smallest tile that is one round: 16 x 2048 x
//   7168 in 16 x 16 5.3 (16 x 32: 6.9, 32 x 64: 9.5), 64 x 2048 x 7168 in 16 x 32 7.0 (32 x 32: 8.4; 16 x 16, two rounds: 9.3), 128 x 2048 x 7168 in 32 x 32 8.5 (32 x 64: 12.0), one
//   row of 7168 x 7168 7.7 (16 x 16: 8.8, 32 x 64: 14.8). Then whole rows of k in tiles that leave few units idle: 32 x 64 up to two a unit, 128 x 7168 x 7168 16.1 (64 x 64: 16.6), 512 x
//   2048 x 7168 16.2 (16.4), but 1024 x 2048 x 7168 19.3 (17.7); 64 x 64 up to four, 4096 x 768 x 2048 9.8 (128 x 128: 11.5), 512 x 7168 x 7168 26.6 (27.9). Behind that whole rounds of
//   256 units count: one of 256 x 256 tiles takes 55 parts of time, of 256 x 128 34, of two 128 x 128 a unit 38. 4096 x 7168 x 7168: 104 in 448 tiles of 256 x 256 (256 x 128: 128, 128 x
//   128: 130), 1024 x 7168 x 7168 32.5 in 224 of 256 x 128 (35.7; 256 x 256: 44.6), 2048 x 7168 x 2048 22.3 (25.4, 26.2), 4096 x 2048 x 2048 15.5 in 256 x 128 (16.2, 20.3).
//   Experts, by slots an expert. Up to 12, while the rows' tiles are two a unit, by waves sharing k: 16 tokens, top 4 of 8, 2048 x 2048 5.9 (32 x 64: 7.5); 64 experts of 7168 rows: 70, 32 x 64
//   50.5. 32 x 64 below 24 slots, or while its tiles are few: 333 tokens, top 2 of 64, 7168 x 2048 90 (64 x 64: 94), 16 slots, 128 experts, 2048 x 768 24.3 (25.9), 128 slots, 8 experts,
//   2048 x 2048 10.6 (10.5). 64 x 64 below 56, or while few: 32 slots, 64 experts, 7168 x 2048 112 (32 x 64: 115, 128 x 128: 121). 128 x 128: 64 slots, 128 experts, 768 x 2048 32.0 (64 x 64:
//   34.9), 128 slots 42.8 (256 x 256: 45.7, 64 x 64: 47.5), 256 slots 62.3 (68.6). 256 x 256 from 352 on: 512 slots 100 (128 x 128: 117), 64 experts, 7168 x 2048 419 (460).
// n_experts 0: one matrix, n its columns; else n slots. reach: the tiles' offsets of gathered columns, 32 bits, hold the columns.
static Mx4Form mx4_form(u32 n_experts, u32 rows, u32 n, bool reach) {
    const auto up = [](u32 x, u32 y) { return (x + y - 1) / y; };
    const auto tiles = [&](u32 bt, u32 br) { return (uint64_t)up(n, bt) * up(rows, br); };
    if (n_experts) {
        const u32 each = n / n_experts, runs = n < n_experts ? n : n_experts;
        if (n <= 32 || !reach || (each <= 12 && (uint64_t)up(rows, 32) * n_experts <= 512)) return kMx4Few16x32;
        // tiles that runs fill, and half a one more for each
        const auto filled = [&](u32 bt) { return (uint64_t)(n / bt + runs / 2) * up(rows, 64); };
        if (each < 24 || filled(32) <= 1200) return kMx4Tile32x64;
        if (each < 56 || filled(64) <= 800) return kMx4Tile64x64;
        return each < 352 ? kMx4Tile128x128 : kMx4Tile256x256;
    }
    if (tiles(16, 16) <= 256) return kMx4Few16x16;
    if (n <= 16 || tiles(16, 32) <= 256) return kMx4Few16x32;
    if (n <= 32 || tiles(32, 32) <= 256) return kMx4Few32x32;
    if (tiles(32, 64) <= 512) return kMx4Tile32x64;
    if (tiles(64, 64) <= 1024) return kMx4Tile64x64;
    const auto rounds = [&](u32 bt, u32 br, u32 at_once) { return (tiles(bt, br) + at_once - 1) / at_once; };
    const uint64_t by256 = 55 * rounds(256, 256, 256), by128 = 34 * rounds(256, 128, 256), by_two = 38 * rounds(128, 128, 512);
    if (by256 <= by128 && by256 <= by_two) return kMx4Tile256x256;
    return by128 <= by_two ? kMx4Tile256x128 : kMx4Tile128x128;
}
static bool mx4_reach(bool gathered, int n_cols, u32 kp) { return !gathered || (uint64_t)n_cols * kp <= 0xffffffffu; }

int mx4_gemm_form(int n_experts, int rows, int k, int n_cols, int n_slots, int top_k) {
    static const struct {
        u32 columns, rows, waves, buffers;
    } of[] = {{16, 16, 8, 4}, {16, 32, 3, 4}, {32, 32, 4, 4}, {32, 64, 2, 2}, {64, 64, 4, 2}, {128, 128, 4, 2}, {256, 128, 8, 2}, {256, 256, 8, 2}};
    const u32 kp = (u32)mx4_row_bytes(k);
    const auto &f = of[mx4_form((u32)n_experts, (u32)rows, (u32)(n_experts ? n_slots : n_cols), mx4_reach(n_experts && top_k > 0, n_cols, kp))];
    return (int)(f.columns | f.rows << 10 | f.waves << 20 | f.buffers << 24);
}

hipError_t mx4_gemm(const Launch &L, const uint8_t *w, const uint8_t *ws, int n_experts, int rows, int k, const uint8_t *q, const uint8_t *qs, int n_cols,
                    const uint32_t *order, const uint32_t *start, int n_slots, int top_k, void *y, int et, int64_t ld) {
    const Mx4Args a = {w, ws, (u32)rows, (u32)mx4_row_bytes(k), (u32)mx4_row_scales(k), q, qs, (u32)n_cols, order, start, (u32)n_slots, (u32)top_k,
                       (u32)n_cols, (u32)n_experts, y, (size_t)ld, et, L.fault, L.layer};
    const u32 n = start ? (u32)n_slots : (u32)n_cols;
    switch (mx4_form(start ? a.n_experts : 0, a.rows, n, mx4_reach(order != nullptr, n_cols, a.kp))) {
    case kMx4Few16x16: return mx4_few_launch<1, 1, 8>(L, a, n);
    case kMx4Few16x32: return mx4_few_launch<2, 1, 3>(L, a, n);
    case kMx4Few32x32: return mx4_few_launch<2, 2, 4>(L, a, n);
    case kMx4Tile32x64: return mx4_tile_launch<32, 64, 1, 2, 0, 2>(L, a, n);
    case kMx4Tile64x64: return mx4_tile_launch<64, 64, 2, 2, 0, 2>(L, a, n);
    case kMx4Tile128x128: return mx4_tile_launch<128, 128, 2, 2, 0, 2>(L, a, n);
    case kMx4Tile256x128: return mx4_tile_launch<256, 128, 4, 2, 2, 2>(L, a, n);
    case kMx4Tile256x256: return mx4_tile_launch<256, 256, 4, 2, 2, 2>(L, a, n);
    }
    return hipErrorInvalidValue;
}

// ------------------------------------------------------------------------------------ a few tokens' experts

// Two launches, three where workgroups share down's lines. The first forms h: a workgroup some rows of gate and of up of an expert that is hit, for up to UC of the tokens that
// picked it. The second forms y: a workgroup 16 R rows of down, for all tokens, over the experts that are hit. Weights are read once by each (once for UC tokens by the first), as lines
// through rings in LDS, and bound both; codes become bf16 values exactly, a few instructions for eight, and the products run on the bf16 matrix instructions, the tokens' values in parts
// that add up to them: x in one of bf16, two of f16, three of f32; h, which is f32 by then, in two parts, 16 bits of mantissa, where y has 8 or 11 (one part of bf16 would leave h the largest
// error of the step: 64 tokens of 7168 x 2048 0.0020 from 64 bits, in two 0.0016, which is y's own rounding; the step 245.6 and 250.5 us), in three where y is f32. (The instructions that take 4-bit codes would want x and h as codes too, or as 8-bit values, whose errors
// a decode step would not have otherwise.)
// On MI355X, us of each launch: 1 token, top 8 of 128, 2048 x 768 bf16 8.4 + 7.6; 16 tokens in f32 40 + 28 + 4.9 for 168 MB of some 66 hit experts' weights (a copy's rate: 32); 64 tokens, 41
// of the 64 experts of 7168 x 2048 here hit, bf16, 149 (4.3 TB/s) + 107 (3.0 TB/s), 44 of them hit, f16 210 + 111, f32 225 + 168.

// What the first launch leaves for the second: the experts that are hit, ascending, and for each and each token the slot that picked it, the first if
// there are several, kMoeNone for none, and its weight, the sum over all of the token's slots of it.
constexpr u32 kMoeExperts = 1024, kMoeNone = 0xffff;
struct MoeTable {
    u32 n_hit, unused[15];
    uint16_t expert[kMoeExperts];
    struct Hit {
        float weight[kMx4MoeTokens];
        uint16_t slot[kMx4MoeTokens];
    } hit[kMoeExperts];
};
struct Mx4Moe {
    const uint8_t *wg, *wgs, *wu, *wus, *wd, *wds;
    u32 n_experts, hidden, ff, n_tokens, top_k;
    const void *x, *resid;
    size_t ld_x, ld_resid, ld_y;
    const u32 *sel;
    const float *w;
    MoeTable *table; // (as many hits as there can be)
    __bf16 *h;       // a slot's parts, rows of ff rounded up to 32 values
    float *partial;  // the second launch's sums where several workgroups share the experts: by workgroup, tokens x hidden rounded up to 4
    void *y;
    GateRule rule;
    u32 *fault, layer;
};
typedef __bf16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2h __attribute__((ext_vector_type(2)));

// A wave's inclusive sums.
__device__ __forceinline__ u32 moe_upto(u32 v) {
    v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);  // one lane up within sixteen
    v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
    v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
    v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
    v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false); // a row's last onto the next
    v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}
// How often the picks name each expert, and the picks; every thread of the workgroup takes part. An id that names no expert is 0xffff, and raised by
// `raise`'s workgroup.
struct MoePicks {
    u32 count[kMoeExperts / 2]; // two to a word
};
template <int T>
__device__ __forceinline__ void moe_picks(const Mx4Moe &a, MoePicks &p, uint16_t *sel, bool raise) {
    const u32 n = a.n_tokens * a.top_k;
    u32 e = threadIdx.x < n ? a.sel[threadIdx.x] : 0u;
    for (u32 i = threadIdx.x; i < kMoeExperts / 2; i += T) p.count[i] = 0;
    __syncthreads();
    for (u32 i = threadIdx.x; i < n;) {
        const bool in = e < a.n_experts;
        sel[i] = in ? (uint16_t)e : (uint16_t)kMoeNone;
        if (in) atomicAdd(&p.count[e >> 1], 1u << (16 * (e & 1)));
        else if (raise && e != 0xffffffffu) bm_raise(a.fault, a.layer, kSiteExpertId);
        if ((i += T) < n) e = a.sel[i];
    }
    __syncthreads();
}
// The experts that are hit, ascending, taken UC picks at a time: the n-th of those shares. False: there are not as many.
struct MoeShare {
    u32 expert, rank, share, n_hit, n_shares; // the expert's number among those that are hit, the share's number among the expert's; of all experts
};
template <int UC>
__device__ __forceinline__ bool moe_nth(const MoePicks &p, u32 n_experts, u32 n, MoeShare &s) {
    const u32 lane = threadIdx.x & 63, words = (n_experts + 127) / 128; // a lane's, two experts each
    u32 word[8], mine = 0;                                              // shares in the upper half, experts in the lower
#pragma unroll
    for (u32 i = 0; i < 8; i++) {
        if (i >= words) break;
        word[i] = p.count[words * lane + i];
        const u32 c0 = word[i] & 0xffffu, c1 = word[i] >> 16;
        mine += ((c0 + UC - 1) / UC + (c1 + UC - 1) / UC) * 0x10000u + (c0 ? 1u : 0u) + (c1 ? 1u : 0u);
    }
    const u32 upto = moe_upto(mine), before = upto - mine, all = (u32)__builtin_amdgcn_readlane((int)upto, 63);
    s.n_hit = all & 0xffffu;
    s.n_shares = all >> 16;
    if (n >= s.n_shares) return false;
    const int at = __builtin_ctzll(__ballot(before >> 16 <= n && n < upto >> 16));
    const u32 start = (u32)__builtin_amdgcn_readlane((int)before, at);
    u32 left = n - (start >> 16);
    s.rank = start & 0xffffu;
#pragma unroll
    for (u32 i = 0; i < 16; i++) {
        const u32 w = (u32)__builtin_amdgcn_readlane((int)word[i / 2], at), c = i & 1 ? w >> 16 : w & 0xffffu, shares = (c + UC - 1) / UC;
        if (left < shares) {
            s.expert = 2 * words * (u32)at + i;
            s.share = left;
            return true;
        }
        left -= shares;
        s.rank += c ? 1u : 0u;
    }
    return false;
}

// Has the compiler take w anew: what is made of it in a loop stays there, and does not wait in registers (eight times as many) for all of them.
__device__ __forceinline__ void moe_anew(v4i &w) { __asm__ volatile("" : "+v"(w)); }
__device__ __forceinline__ u32 moe_anew(u32 v) {
    __asm__ volatile("" : "+v"(v));
    return v;
}
// Eight codes as bf16 values under their scale.
__device__ __forceinline__ v8h moe_codes(u32 word, float s) {
    const v2h p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 1),
              p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 3);
    return v8h{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
// The two halves of a lane's scales of a line as factors.
__device__ __forceinline__ float moe_scale(u32 two, int h) { return bm_bits_f32((h ? two >> 8 : two & 0xffu) << 23); }

__device__ __forceinline__ v8h moe_as_parts(uint4 p) {
    v8h r;
    __builtin_memcpy(&r, &p, 16);
    return r;
}
// The bits of a value's first part, its first eight bits of mantissa, in their upper half: of the next value towards zero, so that what the part leaves of v has v's sign and is not
// zero. An infinity so leaves an infinity, and a code that is one meets no zero but a zero's (and that of a part below bf16's smallest number, of values below 2^-109). What is
// left has no more bits than behind v's own: where v ends with them, the whole of its last one.
__device__ __forceinline__ u32 moe_first_part(float v) { return bm_f32_bits(v) - (v != 0.0f ? 1u : 0u); }
__device__ __forceinline__ __bf16 moe_cut(float v) {
    const uint16_t high = (uint16_t)(moe_first_part(v) >> 16);
    __bf16 r;
    __builtin_memcpy(&r, &high, 2);
    return r;
}
// Eight values in P parts: what a part leaves is the next one's, the last rounded where something is left.
template <int P>
__device__ __forceinline__ void moe_split(const float (&x)[8], v8h (&part)[P]) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; j++) rest[j] = x[j];
#pragma unroll
    for (int p = 0; p < P; p++) {
        if (p == P - 1) { // bf16's own rounding, and f16's second part, to nearest even
#pragma unroll
            for (int j = 0; j < 8; j++) part[p][j] = (__bf16)rest[j];
            break;
        }
        u32 first[8], w[4];
#pragma unroll
        for (int j = 0; j < 8; j++) first[j] = moe_first_part(rest[j]);
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = __builtin_amdgcn_perm(first[2 * j + 1], first[2 * j], 0x07060302u);
        part[p] = moe_as_parts(make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int j = 0; j < 8; j++) rest[j] = __fsub_rn(rest[j], bm_bits_f32(first[j] & 0xffff0000u));
    }
}
template <int ET>
constexpr int kMoeParts = ET == kElemBF16 ? 1 : ET == kElemF16 ? 2 : 3; // of an x
template <int ET>
constexpr int kMoeKept = ET == kElemF32 ? 3 : 2; // of an h: 16 bits of mantissa where y has fewer, f32's where it is f32

// Eight neighbouring values of a row on their way, those behind its end zeros.
template <int ET>
struct MoePiece {
    static constexpr int V = kElemPiece<ET>, N = 8 / V;
    uint4 raw[N];
    __device__ __forceinline__ void ask(const void *x, size_t row, u32 first, u32 k) {
        if (first + 8 <= k) {
#pragma unroll
            for (int n = 0; n < N; n++) raw[n] = elem_piece<ET>(x, row + first + n * V);
            return;
        }
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (first < k) elem_load_some<ET, 8>(x, row + first, k - first, v);
#pragma unroll
        for (int n = 0; n < N; n++) {
            float e[V];
#pragma unroll
            for (int j = 0; j < V; j++) e[j] = v[n * V + j];
            raw[n] = elem_pack<ET>(e);
        }
    }
    __device__ __forceinline__ void parts(v8h (&part)[kMoeParts<ET>]) const {
        if constexpr (ET == kElemBF16) {
            part[0] = moe_as_parts(raw[0]);
        } else {
            float v[8];
#pragma unroll
            for (int n = 0; n < N; n++) {
                float e[V];
                elem_unpack<ET>(raw[n], e);
#pragma unroll
                for (int j = 0; j < V; j++) v[n * V + j] = e[j];
            }
            moe_split<kMoeParts<ET>>(v, part);
        }
    }
};
// A line's values of a token in LDS: a part of 256, sixteen bytes behind every 256 for the banks; what the matrix instructions take begins at moe_at.
constexpr int kMoePart = 544;
__device__ __forceinline__ u32 moe_put(u32 piece) { return 16 * piece + (piece & 16); }
__device__ __forceinline__ u32 moe_at(u32 lane) { return 128 * (lane >> 4) + 16 * (lane >> 5); }
// The sixteen columns of a matrix instruction are P parts of UC tokens each, from column `first` on: where lane column c finds its part of its token in LDS, of rows from
// `row` on; `none`: the row of zeros, for columns that are no token's.
template <int P, int UC>
__device__ __forceinline__ u32 moe_column(u32 c, u32 tokens, u32 row, u32 none, u32 first = 0) {
    static_assert(P * UC <= 16, "a token's parts are columns of one instruction");
    const u32 of = c - first, part = of / UC, token = of - part * UC;
    return part < (u32)P && token < tokens ? (row + token) * (P * kMoePart) + part * kMoePart : none * (P * kMoePart);
}
// What the lane N behind has, of the same sixteen.
template <int N>
__device__ __forceinline__ float moe_behind(float v) {
    return bm_bits_f32((u32)__builtin_amdgcn_update_dpp(0, (int)bm_f32_bits(v), 0x100 | N, 0xf, 0xf, true));
}
// A wave's reads of LDS are done.
__device__ __forceinline__ void lds_read() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0)
    __asm__ volatile("" ::: "memory");
}
// The lowest N bits of m.
template <int N>
__device__ __forceinline__ unsigned long long moe_first(unsigned long long m) {
    unsigned long long rest = m;
#pragma unroll
    for (int j = 0; j < N; j++) rest &= rest - 1;
    return m ^ rest;
}

// A workgroup's share, the n-th: up to UC tokens of an expert. Lane t of every wave has token t's first slot of the expert (kMoeNone: none) and its place among
// the expert's tokens, less those of the shares in front. The first workgroup of an expert leaves its slots for the second launch. 0: there are not as many
// shares; 1: tokens that picked the expert twice have left none for this one; 2: there it is.
struct MoeEntry {
    u32 expert, slot, place, columns, n_shares, rank; // rank: of an expert's first workgroup's first wave
};
template <int UC>
__device__ __forceinline__ int moe_entry(const Mx4Moe &a, const MoePicks &p, const uint16_t *sel, u32 n, MoeEntry &e) {
    const u32 lane = threadIdx.x & 63;
    MoeShare s;
    const bool there = moe_nth<UC>(p, a.n_experts, n, s);
    if (blockIdx.x == 0 && n == 0 && threadIdx.x == 0) a.table->n_hit = s.n_hit;
    if (!there) return 0;
    e.n_shares = s.n_shares;
    e.expert = s.expert;
    e.slot = e.rank = kMoeNone;
    if (lane < a.n_tokens)
        for (u32 i = a.top_k; i-- > 0;)
            if (sel[lane * a.top_k + i] == e.expert) e.slot = lane * a.top_k + i;
    const unsigned long long users = __ballot(e.slot != kMoeNone);
    const u32 n_users = (u32)__builtin_popcountll(users);
    e.place = (u32)__builtin_popcountll(users & ((1ull << lane) - 1)) - s.share * UC;
    if (blockIdx.x == 0 && s.share == 0 && threadIdx.x < 64) {
        if (lane == 0) a.table->expert[s.rank] = (uint16_t)e.expert;
        a.table->hit[s.rank].slot[lane] = (uint16_t)e.slot;
        e.rank = s.rank;
    }
    if (s.share * UC >= n_users) return 1;
    e.columns = min(n_users - s.share * UC, (u32)UC);
    return 2;
}
// Up to sixteen of an expert's tokens, a column each.
struct MoeColumns {
    u32 slot[16], token[16];
};
__device__ __forceinline__ void moe_columns(const MoeEntry &e, MoeColumns &col) {
    if (e.slot == kMoeNone || e.place >= e.columns) return;
    col.slot[e.place] = e.slot;
    col.token[e.place] = threadIdx.x & 63;
}
// And the weights for the second launch. (Asked for behind the first lines, which are waited for anyway.)
__device__ __forceinline__ void moe_weights(const Mx4Moe &a, const uint16_t *sel, const MoeEntry &e) {
    const u32 token = threadIdx.x & 63;
    if (e.rank == kMoeNone || e.slot == kMoeNone) return;
    float by = a.w[e.slot];
    for (u32 s = e.slot + 1; s < (token + 1) * a.top_k; s++)
        if (sel[s] == e.expert) by = __fadd_rn(by, a.w[s]);
    a.table->hit[e.rank].weight[token] = by;
}
// Sixteen rows of h from r0 on, of as many columns as 256 threads have: a thread a value, row threadIdx.x % 16, column threadIdx.x / 16. gate, up: the first of
// the waves' sums, `stride` bytes apart. Where the rows end in the first half of a block its other half becomes zeros.
template <int ET, int NW, int UC>
__device__ __forceinline__ void moe_leave(const Mx4Moe &a, const MoeColumns &col, u32 columns, u32 r0, const uint8_t *gate, const uint8_t *up, u32 stride) {
    constexpr int PH = kMoeKept<ET>;
    static_assert(64 * NW == 256, "sixteen rows by sixteen columns");
    const u32 column = threadIdx.x >> 4, f = r0 + (threadIdx.x & 15), ffp = (a.ff + 31) / 32 * 32;
    if (column >= columns || f >= ffp) return;
    const u32 of = col.slot[column], at = 256 * (threadIdx.x >> 2 & 3) + 16 * column + 4 * (threadIdx.x & 3);
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
        for (int p = 0; p < kMoeParts<ET>; p++) {
            g = __fadd_rn(g, *reinterpret_cast<const float *>(gate + w * stride + at + 16 * p * UC));
            u = __fadd_rn(u, *reinterpret_cast<const float *>(up + w * stride + at + 16 * p * UC));
        }
    bool odd = false;
    float v = 0.0f;
    if (f < a.ff) v = bm_gate_rule(a.rule.act, a.rule.limit, g, u, odd);
    if (odd) bm_raise(a.fault, a.layer, kSiteF32Product);
    __bf16 *to = a.h + (size_t)of * PH * ffp + f;
#pragma unroll
    for (int p = 0; p < PH; p++) {
        const __bf16 part = p == PH - 1 ? (__bf16)v : moe_cut(v);
        v = __fsub_rn(v, (float)part);
        to[(size_t)p * ffp] = part;
        if (r0 + 16 >= a.ff && r0 + 16 < ffp) to[(size_t)p * ffp + 16] = (__bf16)0.0f;
    }
}
constexpr int kMoeUpWaves = 4;

// h of rows of up to 2048 values, two lines a wave at most: a workgroup goes over several tiles of sixteen rows of gate and as many of up, whose lines come through
// a ring of S stages without a stop between the tiles; the tokens' values of a wave's lines stay in LDS. UC tokens a workgroup (an expert with more has several): LDS holds two
// workgroups a unit with 4 of bf16 and f16, 2 of f32, and experts of a decode batch mostly have fewer (16 tokens, top 8 of 128, f32: 40 us; without the products 31).
template <int ET, int S, int UC>
__global__ __launch_bounds__(64 * kMoeUpWaves) __attribute__((amdgpu_waves_per_eu(2))) void k_mx4_moe_up_short(Mx4Moe a, u32 per) {
    constexpr int NW = kMoeUpWaves, P = kMoeParts<ET>, kRow = P * kMoePart, kLoads = 6; // loads of a stage: four of lines, two of scales
    typedef Lines<4> L;
    static_assert(S == 2 || S == 3, "two or three stages");
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], ring2[S > 2 ? NW * L::kStage : 16];
    __shared__ __align__(16) uint8_t sums[NW * 2048], rows[(NW * 2 * UC + 1) * kRow]; // the last row: zeros
    __shared__ MoePicks picks;
    __shared__ MoeColumns col;
    extern __shared__ __align__(16) uint16_t sel[];
    const u32 wave = (u32)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (u32 i = threadIdx.x; i < kRow / 16; i += 64 * NW) reinterpret_cast<uint4 *>(rows + NW * 2 * UC * kRow)[i] = make_uint4(0, 0, 0, 0);
    moe_picks<64 * NW>(a, picks, sel, blockIdx.x == 0 && blockIdx.y == 0);
    for (u32 n = blockIdx.y;; n += gridDim.y) { // (once, where no expert has more than one share)
        u32 lane = threadIdx.x & 63;
        __asm__ volatile("" : "+v"(lane)); // anew for each share: what follows from it does not wait in registers from one to the next
        const u32 c = lane & 15;
        MoeEntry entry;
        const int kind = moe_entry<UC>(a, picks, sel, n, entry);
        if (kind == 0) return;
        if (kind == 1) continue;
        const u32 columns = entry.columns;

        const u32 kp = (a.hidden + 31) / 32 * 16, ks = (a.hidden + 511) / 512 * 16, lines = (kp + 127) / 128, blocks = kp / 16, mine = wave * L::kStage, at = 2 * (lane >> 4);
        const u32 tile0 = blockIdx.x * per, tiles = min(per, (a.ff + 15) / 16 - tile0), each = wave + NW < lines ? 2 : wave < lines ? 1 : 0, items = tiles * each; // this wave's
        const size_t stack = (size_t)entry.expert * a.ff;
        const uint8_t *const gate = a.wg + stack * kp, *const up = a.wu + stack * kp, *const gate_scales = a.wgs + stack * ks, *const up_scales = a.wus + stack * ks;
        L src;
        src.begin(lane);
        u32 s0[2], s1[2], s2[2], asked = 0;
        const auto ask = [&](uint8_t *stage, u32 (&s)[2]) {
            const u32 tile = each == 2 ? asked >> 1 : asked, l = each == 2 && (asked & 1) ? wave + NW : wave, r0 = 16 * (tile0 + tile);
            const u32 mark = min(r0 + c, a.ff - 1) * ks + at + 8 * l; // rows past the last are the last once more, and their values zeros
            s[0] = mx4_two(gate_scales + mark);
            s[1] = mx4_two(up_scales + mark);
#pragma unroll
            for (u32 g = 0; g < 4; g++) src.from[g] = (const int8_t *)(g < 2 ? gate : up) + (size_t)min(r0 + 8 * (g & 1) + (lane >> 3), a.ff - 1) * kp;
            __builtin_amdgcn_sched_barrier(0);
            src.ask(stage + mine, l, kp);
            __builtin_amdgcn_sched_barrier(0);
            asked++;
        };
        moe_columns(entry, col);
        __syncthreads();
        // lanes 0 to 31 take one token's values of a line, eight each, lanes 32 to 63 the next one's
        MoePiece<ET> held[2][UC / 2];
#pragma unroll
        for (u32 i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < UC / 2; j++)
                if (const u32 column = 2 * j + (lane >> 5); i < each && column < columns)
                    held[i][j].ask(a.x, (size_t)col.token[column] * a.ld_x, 256 * (wave + i * NW) + 8 * (lane & 31), a.hidden);
        __builtin_amdgcn_sched_barrier(0);
        if (asked < items) ask(ring0, s0);
        if (asked < items) ask(ring1, s1);
#pragma unroll
        for (u32 i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < UC / 2; j++)
                if (const u32 column = 2 * j + (lane >> 5); i < each && column < columns) {
                    v8h part[P];
                    held[i][j].parts(part);
                    uint8_t *to = rows + ((wave * 2 + i) * UC + column) * kRow + moe_put(lane & 31);
#pragma unroll
                    for (int p = 0; p < P; p++) *reinterpret_cast<v8h *>(to + p * kMoePart) = part[p];
                }
        moe_weights(a, sel, entry);
        v4f acc[2];
        u32 done = 0, tile = 0;
        const auto step = [&](uint8_t *stage, u32 (&s)[2], uint8_t *free, u32 (&next)[2]) {
            const u32 i = each == 2 ? done & 1 : 0, l = wave + i * NW;
            if (done + 1 < items) loads_landed<kLoads>(); // the next stage may be on its way
            else loads_landed<0>();
            if (S > 2 && asked < items) ask(free, next);
            v4i w[2][2];
            float by[2][2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const u32 two = mx4_scales(s[g], 8 * l + at, blocks);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    w[g][h] = mx4_of_line(stage + mine, lane, g, h);
                    by[g][h] = moe_scale(two, h);
                }
            }
            if (S == 2 && asked < items) {
                lds_read(); // the stage is in registers
                ask(stage, s);
            }
            if (i == 0) acc[0] = acc[1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            const uint8_t *row = rows + moe_column<P, UC>(c, columns, (wave * 2 + i) * UC, NW * 2 * UC) + moe_at(lane);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const v8h value = *reinterpret_cast<const v8h *>(row + 16 * j);
#pragma unroll
                for (int g = 0; g < 2; g++) acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(moe_codes((u32)w[g][j / 4][j % 4], by[g][j / 4]), value, acc[g], 0, 0, 0);
            }
            done++;
        };
        // A tile's sums meet: one barrier in front of the sums' reading and one behind it, neither of which waits for lines on their way.
        const auto leave = [&] {
#pragma unroll
            for (int g = 0; g < 2; g++) *reinterpret_cast<v4f *>(sums + wave * 2048 + g * 1024 + 16 * lane) = each ? acc[g] : v4f{0.0f, 0.0f, 0.0f, 0.0f};
            lds_meet();
            moe_leave<ET, NW, UC>(a, col, columns, 16 * (tile0 + tile), sums, sums + 1024, 2048);
            lds_meet();
            tile++;
        };
        const auto turn = [&] { // behind a step: whether its tile is done
            if (each == 1 || !(done & 1)) leave();
        };
        if (each == 0) {
            while (tile < tiles) leave();
        } else {
            for (;;) {
                step(ring0, s0, ring2, s2);
                turn();
                if (done == items) break;
                step(ring1, s1, ring0, s0);
                turn();
                if (done == items) break;
                if (S > 2) {
                    step(ring2, s2, ring1, s1);
                    turn();
                    if (done == items) break;
                }
            }
        }
        if (n + gridDim.y >= entry.n_shares) return;
        __syncthreads();
    }
}

// h. Sixteen rows of gate and as many of up, their lines dealt to the waves, each through three stages, of which two are on
// their way while one is multiplied. A line's values of x come through LDS in parts, the next line's asked for in front of the weights: asked for in the matrix
// instructions' form, each of sixteen requests a line would take the vector cache as long as a line of weights does. (64 tokens, experts of 7168 x 2048: f32 225 us, f16 210 for 44 that are hit; bf16
// 174 for 41, without x 145, several tiles a workgroup instead of one 172.)
template <int ET, int UC>
__global__ __launch_bounds__(64 * kMoeUpWaves) __attribute__((amdgpu_waves_per_eu(2))) void k_mx4_moe_up(Mx4Moe a) {
    constexpr int NW = kMoeUpWaves, P = kMoeParts<ET>, kLoads = 6, kRow = P * kMoePart; // loads of a stage: four of lines, two of scales
    typedef Lines<4> L;
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], ring2[NW * L::kStage];
    __shared__ __align__(16) uint8_t rows[(NW * UC + 1) * kRow]; // the last: zeros
    __shared__ MoePicks picks;
    __shared__ MoeColumns col;
    extern __shared__ __align__(16) uint16_t sel[];
    const u32 wave = (u32)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (u32 i = threadIdx.x; i < kRow / 16; i += 64 * NW) reinterpret_cast<uint4 *>(rows + NW * UC * kRow)[i] = make_uint4(0, 0, 0, 0);
    moe_picks<64 * NW>(a, picks, sel, blockIdx.x == 0 && blockIdx.y == 0);
    for (u32 n = blockIdx.y;; n += gridDim.y) { // (once, where no expert has more than one share)
        u32 lane = threadIdx.x & 63;
        __asm__ volatile("" : "+v"(lane)); // anew for each share: what follows from it does not wait in registers from one to the next
        const u32 c = lane & 15;
        MoeEntry entry;
        const int kind = moe_entry<UC>(a, picks, sel, n, entry);
        if (kind == 0) return;
        if (kind == 1) continue;
        const u32 expert = entry.expert, columns = entry.columns;

        const u32 kp = (a.hidden + 31) / 32 * 16, ks = (a.hidden + 511) / 512 * 16, lines = (kp + 127) / 128, blocks = kp / 16, mine = wave * L::kStage, at = 2 * (lane >> 4);
        const u32 r0 = blockIdx.x * 16;
        L src;
        src.begin(lane);
        const size_t stack = (size_t)expert * a.ff;
        const uint8_t *scales[2];
#pragma unroll
        for (u32 g = 0; g < 4; g++) // rows past the last are the last once more, and their values zeros
            src.from[g] = (const int8_t *)(g < 2 ? a.wg : a.wu) + (stack + min(r0 + 8 * (g & 1) + (lane >> 3), a.ff - 1)) * kp;
#pragma unroll
        for (u32 g = 0; g < 2; g++) scales[g] = (g < 1 ? a.wgs : a.wus) + (stack + min(r0 + c, a.ff - 1)) * ks + at;
        u32 s0[2], s1[2], s2[2];
        const auto ask = [&](uint8_t *stage, u32 (&s)[2], u32 l) {
#pragma unroll
            for (int g = 0; g < 2; g++) s[g] = mx4_two(scales[g] + 8 * l);
            __builtin_amdgcn_sched_barrier(0);
            src.ask(stage + mine, l, kp);
            __builtin_amdgcn_sched_barrier(0);
        };

        moe_columns(entry, col);
        __syncthreads();
        // lanes 0 to 31 take one token's values of a line, eight each, lanes 32 to 63 the next one's
        MoePiece<ET> held[UC / 2];
        size_t row_of[UC / 2];
#pragma unroll
        for (int j = 0; j < UC / 2; j++) row_of[j] = (size_t)col.token[min(2 * j + (lane >> 5), columns - 1)] * a.ld_x;
        const auto fetch = [&](u32 l) {
#pragma unroll
            for (int j = 0; j < UC / 2; j++)
                if (2 * j + (lane >> 5) < columns) held[j].ask(a.x, row_of[j], 256 * l + 8 * (lane & 31), a.hidden);
        };
        const auto put = [&] {
#pragma unroll
            for (int j = 0; j < UC / 2; j++) {
                if (2 * j + (lane >> 5) >= columns) continue;
                v8h part[P];
                held[j].parts(part);
                uint8_t *to = rows + (wave * UC + 2 * j + (lane >> 5)) * kRow + moe_put(lane & 31);
#pragma unroll
                for (int p = 0; p < P; p++) *reinterpret_cast<v8h *>(to + p * kMoePart) = part[p];
            }
        };
        if (wave < lines) fetch(wave);
        __builtin_amdgcn_sched_barrier(0);
        if (wave < lines) ask(ring0, s0, wave);
        if (wave + NW < lines) ask(ring1, s1, wave + NW);
        moe_weights(a, sel, entry);
        v4f acc[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
        const auto step = [&](const uint8_t *stage, u32 (&s)[2], uint8_t *free, u32 (&next)[2], u32 l) {
            if (l + NW < lines) loads_landed<kLoads>(); // the next stage may be on its way; this line's values of x are older than it
            else loads_landed<0>();
            put();
            if (l + NW < lines) fetch(l + NW);
            __builtin_amdgcn_sched_barrier(0);
            if (l + 2 * NW < lines) ask(free, next, l + 2 * NW);
            v4i w[2][2];
            float by[2][2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const u32 two = mx4_scales(s[g], 8 * l + at, blocks);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    w[g][h] = mx4_of_line(stage + mine, lane, g, h);
                    by[g][h] = moe_scale(two, h);
                }
            }
            const uint8_t *row = rows + moe_column<P, UC>(c, columns, wave * UC, NW * UC) + moe_at(lane);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const v8h value = *reinterpret_cast<const v8h *>(row + 16 * i);
#pragma unroll
                for (int g = 0; g < 2; g++) acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(moe_codes((u32)w[g][i / 4][i % 4], by[g][i / 4]), value, acc[g], 0, 0, 0);
            }
        };
        for (u32 l = wave; l < lines;) {
            step(ring0, s0, ring2, s2, l);
            if ((l += NW) >= lines) break;
            step(ring1, s1, ring0, s0, l);
            if ((l += NW) >= lines) break;
            step(ring2, s2, ring1, s1, l);
            l += NW;
        }
        loads_landed<0>();
#pragma unroll
        for (int g = 0; g < 2; g++) *reinterpret_cast<v4f *>(ring0 + mine + g * 1024 + 16 * lane) = acc[g];
        __syncthreads();
        moe_leave<ET, NW, UC>(a, col, columns, r0, ring0, ring0 + 1024, L::kStage);
        if (n + gridDim.y >= entry.n_shares) return;
        __syncthreads();
    }
}

// The same of bf16 rows that lie on 16 bytes and end with a block: their lines and all scales go into LDS as the weights do, two stages of each, and are multiplied as they are. A stage is
// read to registers as a whole and asked for again before it is multiplied, so that values as well as weights are two lines on their way; no load hangs on a condition, since the compiler waits
// by the loads that it can count (of a line's values ASKS loads, two tokens each). Piece p of token c lies at place p ^ c of its line, for the banks. 64 tokens, 41 experts of 7168 x 2048 hit:
// 149 to 153 us, 4.2 TB/s (through registers, a line ahead: 174).
__device__ const uint4 moe_zeros[1] = {};
template <int UC>
__global__ __launch_bounds__(64 * kMoeUpWaves) __attribute__((amdgpu_waves_per_eu(2))) void k_mx4_moe_up_direct(Mx4Moe a) {
    constexpr int NW = kMoeUpWaves, kLoads = 6, kValues = UC * 512; // loads of a stage's weights; bytes of its values
    typedef Lines<4> L;
    static_assert(UC == 8, "a token's number turns the pieces of eight");
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage], rows0[NW * kValues + 512], rows1[NW * kValues + 512]; // the last lines: zeros
    __shared__ __align__(1024) uint8_t marks0[NW * 512], marks1[NW * 512];
    __shared__ MoePicks picks;
    __shared__ MoeColumns col;
    extern __shared__ __align__(16) uint16_t sel[];
    const u32 wave = (u32)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x < 64) reinterpret_cast<uint4 *>((threadIdx.x < 32 ? rows0 : rows1) + NW * kValues)[threadIdx.x & 31] = make_uint4(0, 0, 0, 0);
    moe_picks<64 * NW>(a, picks, sel, blockIdx.x == 0 && blockIdx.y == 0);
    for (u32 n = blockIdx.y;; n += gridDim.y) { // (once, where no expert has more than one share)
        u32 lane = threadIdx.x & 63;
        __asm__ volatile("" : "+v"(lane)); // anew for each share: what follows from it does not wait in registers from one to the next
        const u32 c = lane & 15;
        MoeEntry entry;
        const int kind = moe_entry<UC>(a, picks, sel, n, entry);
        if (kind == 0) return;
        if (kind == 1) continue;
        const u32 columns = entry.columns, asks = (columns + 1) / 2; // of a line's values, two tokens each

        const u32 kp = (a.hidden + 31) / 32 * 16, ks = (a.hidden + 511) / 512 * 16, lines = (kp + 127) / 128, blocks = kp / 16, mine = wave * L::kStage, at = 2 * (lane >> 4);
        const u32 r0 = blockIdx.x * 16;
        const size_t stack = (size_t)entry.expert * a.ff;
        L src;
        src.begin(lane);
        const uint8_t *scales[2];
#pragma unroll
        for (u32 g = 0; g < 4; g++) // rows past the last are the last once more, and their values zeros
            src.from[g] = (const int8_t *)(g < 2 ? a.wg : a.wu) + (stack + min(r0 + 8 * (g & 1) + (lane >> 3), a.ff - 1)) * kp;
#pragma unroll
        for (u32 g = 0; g < 2; g++) scales[g] = (g < 1 ? a.wgs : a.wus) + (stack + min(r0 + c, a.ff - 1)) * ks + (at & 4); // four blocks' at once, of which two are this lane's
        moe_columns(entry, col);
        __syncthreads();
        const uint8_t *of[UC / 2]; // this lane's token of each ask
#pragma unroll
        for (int j = 0; j < UC / 2; j++) of[j] = (const uint8_t *)a.x + (size_t)col.token[min(2 * j + (lane >> 5), columns - 1)] * a.ld_x * 2;
        const auto ask = [&](auto each, uint8_t *stage, uint8_t *rows, uint8_t *marks, u32 l) {
            constexpr int ASKS = decltype(each)::value;
#pragma unroll
            for (int g = 0; g < 2; g++) __builtin_amdgcn_global_load_lds((lds_from *)(scales[g] + 8 * l), (lds_to *)(marks + wave * 512 + 256 * g), 4, 0, 0);
            src.ask(stage + mine, l, kp);
#pragma unroll
            for (int j = 0; j < ASKS; j++) {
                const u32 piece = (lane & 31) ^ (2 * j + (lane >> 5)); // behind the row's end zeros: the codes there are the line's first once more, under the scale 1
                const uint8_t *const from = 8 * l + piece / 4 < blocks ? of[j] + (512 * l + 16 * piece) : (const uint8_t *)moe_zeros;
                __builtin_amdgcn_global_load_lds((lds_from *)from, (lds_to *)(rows + wave * kValues + 1024 * j), 16, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        v4f acc[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
        // kFull: two lines behind this one, the second to be asked for; kNext: one; kLast: none. (No load hangs on a condition: the compiler waits by what it can count.)
        const auto step = [&](auto each, auto place, uint8_t *stage, uint8_t *rows, uint8_t *marks, u32 l) {
            constexpr int ASKS = decltype(each)::value;
            constexpr Mx4Steps STEP = decltype(place)::value;
            loads_landed<STEP == kLast ? 0 : kLoads + ASKS>();
            v4i w[2][2];
            float by[2][2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const u32 two = mx4_scales(*reinterpret_cast<const u32 *>(marks + wave * 512 + 256 * g + 4 * lane) >> 8 * (at & 2) & 0xffff, 8 * l + at, blocks);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    w[g][h] = mx4_of_line(stage + mine, lane, g, h);
                    by[g][h] = moe_scale(two, h);
                }
            }
            const uint8_t *row = rows + (c < columns ? wave * kValues + 512 * c : (u32)(NW * kValues)) + 128 * (lane >> 4);
            v8h value[8];
#pragma unroll
            for (u32 i = 0; i < 8; i++) value[i] = *reinterpret_cast<const v8h *>(row + 16 * (i ^ (c & 7)));
            if (STEP == kFull) {
                lds_read(); // the stage is in registers
                ask(each, stage, rows, marks, l + 2 * NW);
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int g = 0; g < 2; g++) acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(moe_codes((u32)w[g][i / 4][i % 4], by[g][i / 4]), value[i], acc[g], 0, 0, 0);
        };
        const std::integral_constant<Mx4Steps, kFull> full;
        const std::integral_constant<Mx4Steps, kNext> next;
        const std::integral_constant<Mx4Steps, kLast> end;
        const auto run = [&](auto each) {
            ask(each, ring0, rows0, marks0, wave);
            ask(each, ring1, rows1, marks1, wave + NW);
            moe_weights(a, sel, entry);
            u32 l = wave;
            for (; l + 3 * NW < lines; l += 2 * NW) {
                step(each, full, ring0, rows0, marks0, l);
                step(each, full, ring1, rows1, marks1, l + NW);
            }
            if (l + 2 * NW < lines) {
                step(each, full, ring0, rows0, marks0, l);
                step(each, next, ring1, rows1, marks1, l + NW);
                step(each, end, ring0, rows0, marks0, l + 2 * NW);
            } else {
                step(each, next, ring0, rows0, marks0, l);
                step(each, end, ring1, rows1, marks1, l + NW);
            }
        };
        static_assert(UC / 2 == 4, "as many asks");
        if (asks == 1) run(std::integral_constant<int, 1>());
        else if (asks == 2) run(std::integral_constant<int, 2>());
        else if (asks == 3) run(std::integral_constant<int, 3>());
        else run(std::integral_constant<int, 4>());
        loads_landed<0>();
#pragma unroll
        for (int g = 0; g < 2; g++) *reinterpret_cast<v4f *>(ring0 + mine + g * 1024 + 16 * lane) = acc[g];
        __syncthreads();
        moe_leave<kElemBF16, NW, UC>(a, col, columns, r0, ring0, ring0 + 1024, L::kStage);
        if (n + gridDim.y >= entry.n_shares) return;
        __syncthreads();
    }
}

// Four rows' sums of a token onto the residual.
template <int ET>
__device__ __forceinline__ void moe_onto(const Mx4Moe &a, u32 token, u32 row, float (&v)[4]) {
    const u32 have = a.hidden - row;
    if (a.resid)
#pragma unroll
        for (u32 j = 0; j < 4; j++)
            if (j < have) v[j] = __fadd_rn(v[j], elem_load1<ET>(a.resid, token * a.ld_resid + row + j));
    elem_store_some<ET, 4>(a.y, token * a.ld_y + row, have, v);
}
// y. The lines of the experts that are hit, one expert's after another's, are dealt to the waves in stretches, each through two stages of 16 R rows; the
// waves' sums, NT tiles of sixteen tokens, meet in LDS. A line's values of h come through LDS too, UC tokens' at a time and the next line's asked for in front of the
// weights. The tokens of an expert stand side by side in a matrix instruction's columns, and their sums change to the tokens' own places when the expert's lines end: by
// the tokens' places from the start a line would be multiplied for every tile of sixteen that has one of them (64 tokens, bf16, h in one part: 113 us for 97; in two, 107). gridDim.y workgroups share the
// lines: where they are several, a third launch adds their sums.
template <int ET, int NW, int R, int UC, int NT>
__global__ __launch_bounds__(64 * NW) void k_mx4_moe_down(Mx4Moe a) {
    constexpr int PH = kMoeKept<ET>, NL = (PH + 1) / 2, CH = R == 1 ? 2 : 1; // requests of a token's values; chains of products
    constexpr int kGroups = 16 / (PH * UC), kTokens = kGroups * UC;          // of UC tokens in an instruction's columns
    constexpr int kLoads = 3 * R, kRow = PH * kMoePart;                      // loads of a stage
    typedef Lines<2 * R> L;
    __shared__ __align__(1024) uint8_t ring0[NW * L::kStage], ring1[NW * L::kStage];
    __shared__ __align__(16) uint8_t rows[(NW * UC + 1) * kRow]; // the last: zeros
    __shared__ __align__(16) uint16_t list[kMoeExperts];
    const u32 lane = threadIdx.x & 63, wave = (u32)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = 2 * (lane >> 4), c = lane & 15;
    const u32 n_hit = a.table->n_hit;
    for (u32 i = threadIdx.x; 2 * i < a.n_experts; i += 64 * NW) reinterpret_cast<u32 *>(list)[i] = reinterpret_cast<const u32 *>(a.table->expert)[i];
    for (u32 i = threadIdx.x; i < kRow / 16; i += 64 * NW) reinterpret_cast<uint4 *>(rows + NW * UC * kRow)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();

    const u32 kp = (a.ff + 31) / 32 * 16, ks = (a.ff + 511) / 512 * 16, lines = (kp + 127) / 128, blocks = kp / 16, mine = wave * L::kStage;
    const u32 r0 = blockIdx.x * (16 * R), ffp = (a.ff + 31) / 32 * 32, shares = NW * gridDim.y, share = NW * blockIdx.y + wave, items = n_hit * lines;
    const u32 q0 = items * share / shares, q1 = items * (share + 1) / shares;
    L src;
    src.begin(lane);
    u32 n = q0 / lines, l = q0 - n * lines, ask_n = n, ask_l = l, ask_q = q0;
    u32 s0[R], s1[R];
    const auto ask = [&](uint8_t *stage, u32 (&s)[R]) {
        const size_t row = (size_t)(u32)__builtin_amdgcn_readfirstlane(list[ask_n]) * a.hidden + r0;
        const uint8_t *const codes = a.wd + row * kp, *const scales = a.wds + row * ks + 8 * ask_l;
        const u32 of = moe_anew(lane), last = a.hidden - 1 - r0; // rows past the last are the last once more, and not stored
#pragma unroll
        for (u32 g = 0; g < R; g++) s[g] = mx4_two(scales + (min(16 * g + (of & 15), last) * ks + 2 * (of >> 4)));
#pragma unroll
        for (u32 g = 0; g < 2 * R; g++) src.from[g] = (const int8_t *)codes + min(8 * g + (of >> 3), last) * kp;
        __builtin_amdgcn_sched_barrier(0);
        src.ask(stage + mine, ask_l, kp);
        __builtin_amdgcn_sched_barrier(0);
        ask_q++;
        if (++ask_l == lines) ask_l = 0, ask_n++;
    };

    // The tokens of an expert: lane t's slot and weight (of up to 16 tokens: lane t % 16's), and those that have one, as bits.
    u32 slot = kMoeNone, next_slot = kMoeNone;
    float weight = 0.0f, next_weight = 0.0f;
    unsigned long long users = 0;
    const u32 part_at = (lane >> 5) * ffp + 8 * (lane & 31), put_at = (lane >> 5) * kMoePart + moe_put(lane & 31);
    uint4 held[UC * NL];
    // Line `line` of the tokens that `some` holds, the first UC of them.
    const auto fetch = [&](unsigned long long some, u32 slots, u32 line) {
#pragma unroll
        for (int j = 0; j < UC; j++) {
            if (some) {
                const u32 of = (u32)__builtin_amdgcn_readlane((int)slots, __builtin_ctzll(some));
                const __bf16 *h = a.h + (size_t)of * PH * ffp + 256 * line + moe_anew(part_at);
                const bool there = 8 * line + (lane & 31) / 4 < blocks;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (there && (2 * i + 1 < PH || lane < 32)) v = *reinterpret_cast<const uint4 *>(h + (size_t)(2 * i) * ffp);
                    held[j * NL + i] = v;
                }
            }
            some &= some - 1;
        }
    };
    const auto put = [&](unsigned long long some) {
#pragma unroll
        for (int j = 0; j < UC; j++) {
            if (some)
#pragma unroll
                for (int i = 0; i < NL; i++)
                    if (2 * i + 1 < PH || lane < 32) *reinterpret_cast<uint4 *>(rows + (wave * UC + j) * kRow + 2 * i * kMoePart + put_at) = held[j * NL + i];
            some &= some - 1;
        }
    };
    v4f acc[NT][R];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < R; r++) acc[t][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    v4f sum[R][CH];
    const auto clear = [&] {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < CH; i++) sum[r][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();
    // The sums of the tokens `here`, which have columns by their order, under their weights onto what these tokens have. What the others have stays: zeros times a NaN
    // scale or an infinity are no zeros.
    const auto count = [&](unsigned long long here) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const u32 some = (u32)(here >> (16 * t)) & 0xffffu;
            if (NT > 1 && some == 0) continue;
            const bool user = some >> c & 1;
            const u32 rank = (u32)__builtin_popcountll(here & ((1ull << (16 * t)) - 1)) + (u32)__builtin_popcount(some & ((1u << c) - 1)), group = rank / UC;
            const int from = (int)((lane & 48) + group * (PH * UC) + (rank - group * UC));
            const float by = NT == 1 ? weight : __shfl(weight, 16 * t + c);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float mine = CH > 1 ? __fadd_rn(sum[r][0][i], sum[r][CH - 1][i]) : sum[r][0][i];
                    float v = mine;
                    v = __fadd_rn(v, moe_behind<UC>(mine));
                    if (PH > 2) v = __fadd_rn(v, moe_behind<2 * UC>(mine));
                    v = __shfl(v, from);
                    acc[t][r][i] = user ? __fmaf_rn(by, v, acc[t][r][i]) : acc[t][r][i];
                }
        }
        clear();
    };
    const auto step = [&](uint8_t *stage, u32 (&s)[R], u32 q) {
        if (q + 1 < q1) loads_landed<kLoads>(); // the next stage may be on its way; this line's values of h are older than it
        else loads_landed<0>();
        put(moe_first<UC>(users));
        const bool turn = l + 1 == lines;
        const unsigned long long next_users = turn ? __ballot(next_slot != kMoeNone) : users;
        if (q + 1 < q1) fetch(moe_first<UC>(next_users), turn ? next_slot : slot, turn ? 0 : l + 1);
        const bool more = turn && n + 2 < n_hit;
        const u32 of = moe_anew(lane), after = more ? a.table->hit[n + 2].slot[of] : kMoeNone;
        const float after_weight = more ? a.table->hit[n + 2].weight[NT == 1 ? of & 15 : of] : 0.0f;
        __builtin_amdgcn_sched_barrier(0);
        v4i w[R][2];
        float by[R][2];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const u32 two = mx4_scales(s[r], 8 * l + at, blocks);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                w[r][h] = mx4_of_line(stage + mine, lane, r, h);
                by[r][h] = moe_scale(two, h);
            }
        }
        if (ask_q < q1) {
            lds_read(); // the stage is in registers
            ask(stage, s);
        }
        // The expert's tokens, as many as have columns of their own at a time: where that is all of them, their sums stay over the expert's lines.
        for (unsigned long long rest = users, first = moe_first<UC>(users);;) {
            unsigned long long here = rest;
            if (__builtin_popcountll(rest) > kTokens) here = moe_first<kTokens>(rest);
            unsigned long long some = moe_first<UC>(here), left = here ^ some;
            const bool groups = left != 0;
            for (u32 column = 0;; column += PH * UC) {
                if (some != first) { // (the values of the next line that are held are in LDS only after these)
                    uint4 keep[UC * NL];
#pragma unroll
                    for (int i = 0; i < UC * NL; i++) keep[i] = held[i];
                    fetch(some, slot, l);
                    put(some);
#pragma unroll
                    for (int i = 0; i < UC * NL; i++) held[i] = keep[i];
                }
#pragma unroll
                for (int r = 0; r < R; r++) moe_anew(w[r][0]), moe_anew(w[r][1]);
                const uint8_t *row = rows + moe_column<PH, UC>(c, (u32)__builtin_popcountll(some), wave * UC, NW * UC, column) + moe_at(lane);
                v4f others[R][CH]; // what the other groups' columns have: an infinite code would make NaN of the zeros that stand there now
                if constexpr (kGroups > 1) {
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int i = 0; i < CH; i++) others[r][i] = sum[r][i];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const v8h value = *reinterpret_cast<const v8h *>(row + 16 * i);
#pragma unroll
                    for (int r = 0; r < R; r++) sum[r][i % CH] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(moe_codes((u32)w[r][i / 4][i % 4], by[r][i / 4]), value, sum[r][i % CH], 0, 0, 0);
                }
                if constexpr (kGroups > 1) {
                    if (groups)
#pragma unroll
                        for (int r = 0; r < R; r++)
#pragma unroll
                            for (int i = 0; i < CH; i++) sum[r][i] = c - column < (u32)(PH * UC) ? sum[r][i] : others[r][i];
                }
                if (!left) break;
                some = moe_first<UC>(left);
                left ^= some;
            }
            rest ^= here;
            if (turn || q + 1 == q1 || here != users) count(here);
            if (!rest) break;
        }
        if (turn) {
            l = 0, n++;
            slot = next_slot, users = next_users, next_slot = after;
            weight = next_weight, next_weight = after_weight;
        } else {
            l++;
        }
    };
    if (q0 < q1) {
        slot = a.table->hit[n].slot[lane], weight = a.table->hit[n].weight[NT == 1 ? c : lane];
        if (n + 1 < n_hit) next_slot = a.table->hit[n + 1].slot[lane], next_weight = a.table->hit[n + 1].weight[NT == 1 ? c : lane];
        users = __ballot(slot != kMoeNone);
        fetch(moe_first<UC>(users), slot, l);
        __builtin_amdgcn_sched_barrier(0);
        ask(ring0, s0);
        if (ask_q < q1) ask(ring1, s1);
        for (u32 q = q0;;) {
            step(ring0, s0, q);
            if (++q == q1) break;
            step(ring1, s1, q);
            if (++q == q1) break;
        }
    }
    loads_landed<0>();
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int r = 0; r < R; r++) *reinterpret_cast<v4f *>(ring0 + mine + r * 1024 + 16 * lane) = acc[t][r];
        __syncthreads();
        const u32 token = 16 * t + c, row = r0 + 16 * wave + 4 * (lane >> 4);
        if (wave < R && token < a.n_tokens && row < a.hidden) {
            const v4f sum = mx4_join<NW, L>(ring0, wave, lane);
            float v[4] = {sum[0], sum[1], sum[2], sum[3]};
            if (gridDim.y > 1) *reinterpret_cast<v4f *>(a.partial + ((size_t)blockIdx.y * a.n_tokens + token) * ((a.hidden + 3) / 4 * 4) + row) = sum;
            else moe_onto<ET>(a, token, row, v);
        }
        __syncthreads();
    }
}
constexpr u32 kMoeSharers = 8;
// The workgroups' sums, in their order.
template <int ET>
__global__ __launch_bounds__(256) void k_mx4_moe_join(Mx4Moe a, u32 n) {
    const u32 quads = (a.hidden + 3) / 4, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= quads * a.n_tokens) return;
    v4f part[kMoeSharers], sum; // all asked for at once, the last as often as there are fewer
#pragma unroll
    for (u32 z = 0; z < kMoeSharers; z++) part[z] = *reinterpret_cast<const v4f *>(a.partial + ((size_t)min(z, n - 1) * quads * a.n_tokens + i) * 4);
    sum = part[0];
#pragma unroll
    for (u32 z = 1; z < kMoeSharers; z++)
        if (z < n) sum += part[z];
    float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    moe_onto<ET>(a, i / quads, 4 * (i % quads), v);
}

static u32 moe_hits(int n_tokens, int top_k, int n_experts) { return (u32)std::min(n_tokens * top_k, n_experts); }
template <int ET, int UC>
static void moe_up(const Launch &L, const Mx4Moe &a) {
    hipLaunchKernelGGL((k_mx4_moe_up<ET, UC>), dim3((a.ff + 15) / 16, moe_hits(a.n_tokens, a.top_k, a.n_experts)), dim3(64 * kMoeUpWaves),
                       (a.n_tokens * a.top_k * 2 + 15) & ~15u, L.stream, a);
}
template <int ET, int S, int UC>
static void moe_up_short(const Launch &L, const Mx4Moe &a) {
    const u32 tiles = (a.ff + 15) / 16, hits = moe_hits(a.n_tokens, a.top_k, a.n_experts), per = std::max(1u, tiles * hits / 1536);
    hipLaunchKernelGGL((k_mx4_moe_up_short<ET, S, UC>), dim3((tiles + per - 1) / per, hits), dim3(64 * kMoeUpWaves), (a.n_tokens * a.top_k * 2 + 15) & ~15u, L.stream, a, per);
}
// Workgroups that share the lines of down's experts: where its rows are few, as many as fill the card (two a slot of a token at most: what the scratch holds).
static u32 moe_sharers(int top_k, int hidden) { return (u32)std::max(1, std::min({(int)kMoeSharers, 2 * top_k, 256 * 32 / hidden})); }
template <int ET, int NW, int R, int UC, int NT>
static hipError_t moe_down(const Launch &L, const Mx4Moe &a, u32 sharers) {
    hipLaunchKernelGGL((k_mx4_moe_down<ET, NW, R, UC, NT>), dim3((a.hidden + 16 * R - 1) / (16 * R), sharers), dim3(64 * NW), 0, L.stream, a);
    const hipError_t e = hipGetLastError();
    if (sharers == 1 || e != hipSuccess) return e;
    hipLaunchKernelGGL((k_mx4_moe_join<ET>), dim3(((a.hidden + 3) / 4 * a.n_tokens + 255) / 256), dim3(256), 0, L.stream, a, sharers);
    return hipGetLastError();
}
// Up's lines stay with their values where a wave has two at most: 16 tokens in f32, rows of 2048, 40 us (46 against 50 a line at a time before a token's parts were columns of one instruction), one token in
// bf16 8.2 (8.8). Down in 32 rows a workgroup where these fill the card, alone or shared (16 tokens, 2048 rows, f32: four sharers 28 and 4.9 for their sums; when these took 29, of 16 rows a workgroup 33, unshared 42), else 16. The whole step of 64 tokens, 7168 rows, bf16: 250.5 with 12
// waves, 272 with 14 that have the values of three tokens, 284 with 8; f16 302, 324, 336.
template <int ET, int NT>
static hipError_t moe_launch(const Launch &L, const Mx4Moe &a) {
    constexpr int P = kMoeParts<ET>;
    if (a.hidden <= 256 * 2 * kMoeUpWaves) moe_up_short<ET, P == 1 ? 3 : 2, P == 3 ? 2 : 4>(L, a);
    else if (P == 1 && a.hidden % 32 == 0 && a.ld_x % 8 == 0 && ((uintptr_t)a.x & 15) == 0)
        hipLaunchKernelGGL((k_mx4_moe_up_direct<8>), dim3((a.ff + 15) / 16, moe_hits(a.n_tokens, a.top_k, a.n_experts)), dim3(64 * kMoeUpWaves),
                           (a.n_tokens * a.top_k * 2 + 15) & ~15u, L.stream, a);
    else moe_up<ET, P == 1 ? 8 : 4>(L, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int NW = kMoeKept<ET> == 3 ? 8 : 12, UC = 4; // what LDS holds: their lines, and the values of UC tokens each
    const u32 items = moe_hits(a.n_tokens, a.top_k, a.n_experts) * ((a.ff + 255) / 256);
    const u32 sharers = std::min(moe_sharers(a.top_k, a.hidden), items / (4 * NW));
    if (sharers > 1) return moe_down<ET, NW, 2, UC, NT>(L, a, sharers);
    if (a.hidden < 4096) return moe_down<ET, 16, 1, P == 3 ? 3 : 4, NT>(L, a, 1);
    return moe_down<ET, NW, 2, UC, NT>(L, a, 1);
}

static size_t moe_table(int n_tokens, int top_k) { return offsetof(MoeTable, hit) + (size_t)moe_hits(n_tokens, top_k, kMoeExperts) * sizeof(MoeTable::Hit); }
static size_t moe_h(int n_tokens, int top_k, int ff) { return (size_t)n_tokens * top_k * 3 * ((ff + 31) / 32 * 32) * 2; }
size_t mx4_moe_work(int n_tokens, int top_k, int hidden, int ff) {
    const u32 sharers = moe_sharers(top_k, hidden);
    return moe_table(n_tokens, top_k) + moe_h(n_tokens, top_k, ff) + (sharers > 1 ? (size_t)sharers * n_tokens * ((hidden + 3) / 4 * 4) * sizeof(float) : 0);
}

hipError_t mx4_moe(const Launch &L, const Mx4Stack &g, const Mx4Stack &u, const Mx4Stack &d, int n_experts, int hidden, int ff, const void *x, int et,
                   int64_t ld_x, int n_tokens, const uint32_t *sel, const float *w, int top_k, const void *resid, int64_t ld_resid, void *y, int64_t ld_y,
                   void *work) {
    const Mx4Moe a = {g.w, g.scales, u.w, u.scales, d.w, d.scales, (u32)n_experts, (u32)hidden, (u32)ff, (u32)n_tokens, (u32)top_k, x, resid, (size_t)ld_x,
                      (size_t)ld_resid, (size_t)ld_y, sel, w, (MoeTable *)work, (__bf16 *)((uint8_t *)work + moe_table(n_tokens, top_k)),
                      (float *)((uint8_t *)work + moe_table(n_tokens, top_k) + moe_h(n_tokens, top_k, ff)), y, L.rule, L.fault,
                      L.layer};
    const bool few = n_tokens <= 16;
    if (et == kElemF32) return few ? moe_launch<kElemF32, 1>(L, a) : moe_launch<kElemF32, 4>(L, a);
    if (et == kElemF16) return few ? moe_launch<kElemF16, 1>(L, a) : moe_launch<kElemF16, 4>(L, a);
    return few ? moe_launch<kElemBF16, 1>(L, a) : moe_launch<kElemBF16, 4>(L, a);
}

} // namespace bmk
