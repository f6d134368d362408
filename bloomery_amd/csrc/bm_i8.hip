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

namespace bmk {

typedef int v4i __attribute__((ext_vector_type(4)));

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

// T threads a row (a wave, or the workgroup), CH pieces of eight values a thread held in registers between the maximum and the codes; CH = 0: a
// row of any length, read twice (the second time from the cache).
template <int ET, bool GLU, int T, int CH>
__global__ __launch_bounds__(256) void k_i8_quantize(QuantArgs a) {
    __shared__ u32 top[4];
    const u32 lane = threadIdx.x % T, row = blockIdx.x * (256 / T) + threadIdx.x / T;
    const u32 m = a.live ? min(a.m, *a.live) : a.m;
    if (row >= m) return; // whole waves (T = 64) or the workgroup (T = 256)
    float v[CH ? CH : 1][8];
    u32 most = 0;
    bool odd = false;
    const u32 pieces = a.kp / 8;
    if constexpr (CH > 0) {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const u32 c = lane + i * T;
            if (c < pieces) quant_values<ET, GLU>(a, row, 8 * c, v[i], odd);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] = 0.0f;
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
    if constexpr (T == 256) {
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = most;
        __syncthreads();
        most = max(max(top[0], top[1]), max(top[2], top[3]));
    }
    // positive floats order as their bits; infinities and NaN lie on top
    const bool bad = most >= 0x7f800000u;
    const float s = bad ? bm_bits_f32(0x7fc00000u) : __fdiv_rn(bm_bits_f32(most), 127.0f);
    if (lane == 0) {
        a.scales[row] = s;
        if (bad) bm_raise(a.fault, a.layer, kSiteQuantColumn);
    }
    // small scales, whose reciprocal could overflow, go up by 2^100 with their values (exactly)
    const float up = s < 0x1p-64f ? 0x1p100f : 1.0f, su = s * up, inv = __fdiv_rn(1.0f, su);
    const bool zero = bad || most == 0 || s == 0.0f;
    int8_t *out = a.codes + (size_t)row * a.kp;
#pragma unroll
    for (int i = 0; i < (CH ? CH : 1); i++)
        for (u32 c = lane + (u32)i * T; c < pieces; c += CH ? pieces : T) {
            if constexpr (CH == 0) quant_values<ET, GLU>(a, row, 8 * c, v[0], odd);
            u32 word[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++) word[j / 4] |= ((u32)(zero ? 0 : i8_code(v[i][j] * up, su, inv)) & 0xffu) << (8 * (j % 4));
            *reinterpret_cast<uint2 *>(out + 8 * c) = make_uint2(word[0], word[1]);
        }
}

template <int ET, bool GLU>
static void quant_launch(const Launch &L, const QuantArgs &a) {
    const dim3 block(256), wave_a_row((a.m + 3) / 4), group_a_row(a.m);
    if (a.kp <= 512) hipLaunchKernelGGL((k_i8_quantize<ET, GLU, 64, 1>), wave_a_row, block, 0, L.stream, a);
    else if (a.kp <= 1024) hipLaunchKernelGGL((k_i8_quantize<ET, GLU, 64, 2>), wave_a_row, block, 0, L.stream, a);
    else if (a.kp <= 2048) hipLaunchKernelGGL((k_i8_quantize<ET, GLU, 256, 1>), group_a_row, block, 0, L.stream, a);
    else if (a.kp <= 4096) hipLaunchKernelGGL((k_i8_quantize<ET, GLU, 256, 2>), group_a_row, block, 0, L.stream, a);
    else if (a.kp <= 8192) hipLaunchKernelGGL((k_i8_quantize<ET, GLU, 256, 4>), group_a_row, block, 0, L.stream, a);
    else hipLaunchKernelGGL((k_i8_quantize<ET, GLU, 256, 0>), group_a_row, block, 0, L.stream, a);
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

// Four neighbouring values of an output row from r on, those below `rows`.
__device__ __forceinline__ void i8_store4(const I8Args &a, u32 j, u32 r, const float (&v)[4]) {
    const size_t at = (size_t)j * a.ld + r;
    const u32 have = a.rows - r;
    if (a.et == kElemF32) elem_store_some<kElemF32, 4>(a.y, at, have, v);
    else if (a.et == kElemF16) elem_store_some<kElemF16, 4>(a.y, at, have, v);
    else elem_store_some<kElemBF16, 4>(a.y, at, have, v);
}

// Few columns a matrix: 16 R rows a workgroup against 16 C columns, its NW waves dealing the row's 64-byte steps among them. Weights go
// from memory to registers in the form v_mfma_i32_16x16x64_i8 takes them (lane l: row l % 16, bytes 16 (l / 16) .. + 15 of the step), each once;
// the columns come from the cache. The waves' sums meet in LDS as integers.
template <int R, int C, int NW>
__global__ __launch_bounds__(64 * NW) void k_i8_few(I8Args a) {
    __shared__ v4i part[NW][R * C][64];
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x;
    I8Run run;
    if (!i8_run(a, blockIdx.y, run)) return;
    const u32 r0 = blockIdx.x * (16 * R), steps = (a.kp + 63) / 64;
    const int8_t *wp[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const u32 row = r0 + 16 * r + (lane & 15);
        wp[r] = run.w + (size_t)(row < a.rows ? row : a.rows - 1) * a.kp; // rows past the last are not stored
    }
    for (u32 t0 = run.j0 + blockIdx.z * (16 * C); t0 < run.j1; t0 += gridDim.z * (16 * C)) {
        const int8_t *qp[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const u32 j = t0 + 16 * c + (lane & 15);
            bool bad;
            qp[c] = a.q + (size_t)i8_column(a, j < run.j1 ? j : run.j1 - 1, bad) * a.kp;
        }
        v4i acc[R][C];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) acc[r][c] = v4i{0, 0, 0, 0};
#pragma unroll 2
        for (u32 s = wave; s < steps; s += NW) {
            const u32 at = 64 * s + 16 * (lane >> 4);
            const bool in = at < a.kp; // a piece past the row: any of the row's bytes against zeros
            const u32 off = in ? at : 0;
            v4i A[R], B[C];
#pragma unroll
            for (int r = 0; r < R; r++) A[r] = *reinterpret_cast<const v4i *>(wp[r] + off);
#pragma unroll
            for (int c = 0; c < C; c++) {
                B[c] = *reinterpret_cast<const v4i *>(qp[c] + off);
                if (!in) B[c] = v4i{0, 0, 0, 0};
            }
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int c = 0; c < C; c++) acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[r], B[c], acc[r][c], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < C; c++) part[wave][r * C + c][lane] = acc[r][c];
        __syncthreads();
        // four rows (4 (l / 16) ..) of one column (l % 16) a lane of a tile
        for (u32 i = tid; i < R * C * 64; i += 64 * NW) {
            const u32 tile = i / 64, l = i % 64;
            v4i sum = part[0][tile][l];
#pragma unroll
            for (int w = 1; w < NW; w++) sum += part[w][tile][l];
            const u32 j = t0 + 16 * (tile % C) + (l & 15), row = r0 + 16 * (tile / C) + 4 * (l >> 4);
            if (j < run.j1 && row < a.rows) {
                bool bad;
                const u32 col = i8_column(a, j, bad);
                if (bad) bm_raise(a.fault, a.layer, kSiteExpertId);
                const float s = bad ? bm_bits_f32(0x7fc00000u) : a.qs[col];
                float v[4];
#pragma unroll
                for (int x = 0; x < 4; x++) v[x] = __fmul_rn(__fmul_rn((float)sum[x], s), run.ws[row + x < a.rows ? row + x : row]);
                i8_store4(a, j, row, v);
            }
        }
        __syncthreads();
    }
}

hipError_t i8_gemm(const Launch &L, const int8_t *w, const float *ws, int n_experts, int rows, int k, const int8_t *q, const float *qs, int n_cols,
                   const uint32_t *order, const uint32_t *start, int n_slots, int top_k, void *y, int et, int64_t ld) {
    const I8Args a = {w, ws, (u32)rows, (u32)i8_row_bytes(k), q, qs, (u32)n_cols, order, start, (u32)n_slots, (u32)top_k, (u32)n_cols, (u32)n_experts,
                      y, (size_t)ld, et, L.fault, L.layer};
    const u32 entries = start ? (u32)n_slots : (u32)n_cols;
    const u32 z = start ? 1u : (entries + 31) / 32;
    hipLaunchKernelGGL((k_i8_few<1, 2, 8>), dim3(((u32)rows + 15) / 16, start ? (u32)n_experts : 1u, z < 65535u ? z : 65535u), dim3(512), 0, L.stream, a);
    return hipGetLastError();
}

} // namespace bmk
