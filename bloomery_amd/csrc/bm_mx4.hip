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

// A wave takes sixteen blocks of a row, sixteen bytes of its scales: a lane eight values, four lanes a block.
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
    u32 most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = max(most, bm_f32_bits(v[j]) & 0x7fffffffu);
    most = quad_max(most) >> 23; // biased exponent
    const bool bad = most == 255;
    const u32 scale = bad ? 255 : most > 2 ? most - 2 : 0;
    if ((lane & 3) == 0) {
        a.scales[(size_t)row * a.ks + block] = (uint8_t)scale;
        if (bad) bm_raise(a.fault, a.layer, kSiteQuantColumn);
    }
    if (16 * block >= a.kp) return;
    u32 word = 0;
    const float s = bm_bits_f32(scale << 23); // the conversion takes the exponent's bits, 0 for 2^-127
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], s, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], s, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], s, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], s, 3);
    *reinterpret_cast<u32 *>(a.codes + (size_t)row * a.kp + c / 2) = bad ? 0u : word;
}

// Eight codes as values.
__device__ __forceinline__ void mx4_values(u32 word, u32 scale, float (&v)[8]) {
    const float s = bm_bits_f32(scale << 23);
    const v2f p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 1),
              p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, 3);
    v[0] = p0[0], v[1] = p0[1], v[2] = p1[0], v[3] = p1[1], v[4] = p2[0], v[5] = p2[1], v[6] = p3[0], v[7] = p3[1];
}

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

// Sixteen rows by sixteen columns, 128 values of k: lane l holds a block of row (column) l % 16, four blocks in turn, and its scale in the
// lowest byte; it gets column l % 16, rows 4 (l / 16) .. + 3.
__device__ __forceinline__ v4f mx4_mfma(v4i w, v4i q, v4f acc, u32 ws, u32 qs) {
    const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {q[0], q[1], q[2], q[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, (int)ws, 0, (int)qs);
}

// A wave sixteen rows and sixteen columns, straight from memory.
__global__ __launch_bounds__(256) void k_mx4_gemm(Mx4Args a) {
    const u32 lane = threadIdx.x & 63, r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, blocks = a.kp / 16;
    Mx4Run run;
    if (!mx4_run(a, blockIdx.y, run) || r0 >= a.rows) return;
    const size_t row = min(r0 + (lane & 15), a.rows - 1);
    for (u32 t0 = run.j0 + blockIdx.z * 16; t0 < run.j1; t0 += gridDim.z * 16) {
        bool bad;
        const size_t col = run_column(a, min(t0 + (lane & 15), run.j1 - 1), bad);
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (u32 b0 = 0; b0 < blocks; b0 += 4) {
            const u32 b = b0 + (lane >> 4);
            v4i w = {0, 0, 0, 0}, q = {0, 0, 0, 0};
            u32 ws = 127, qs = 127;
            if (b < blocks) {
                w = *reinterpret_cast<const v4i *>(run.w + row * a.kp + 16 * b);
                q = *reinterpret_cast<const v4i *>(a.q + col * a.kp + 16 * b);
                ws = run.ws[row * a.ks + b], qs = a.qs[col * a.ks + b];
            }
            acc = mx4_mfma(w, q, acc, ws, qs);
        }
        const u32 j = t0 + (lane & 15), r = r0 + 4 * (lane >> 4);
        if (j >= run.j1 || r >= a.rows) continue;
        if (bad) bm_raise(a.fault, a.layer, kSiteExpertId);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = bad ? bm_bits_f32(0x7fc00000u) : acc[i];
        run_store4(a, j, r, v);
    }
}

hipError_t mx4_gemm(const Launch &L, const uint8_t *w, const uint8_t *ws, int n_experts, int rows, int k, const uint8_t *q, const uint8_t *qs, int n_cols,
                    const uint32_t *order, const uint32_t *start, int n_slots, int top_k, void *y, int et, int64_t ld) {
    const Mx4Args a = {w, ws, (u32)rows, (u32)mx4_row_bytes(k), (u32)mx4_row_scales(k), q, qs, (u32)n_cols, order, start, (u32)n_slots, (u32)top_k,
                       (u32)n_cols, (u32)n_experts, y, (size_t)ld, et, L.fault, L.layer};
    const u32 z = start ? 1u : (a.m + 15) / 16;
    hipLaunchKernelGGL(k_mx4_gemm, dim3((a.rows + 63) / 64, start ? a.n_experts : 1u, z < 65535u ? z : 65535u), dim3(256), 0, L.stream, a);
    return hipGetLastError();
}

hipError_t mx4_gemm_x(const Launch &L, const uint8_t *w, const uint8_t *ws, int rows, int k, const void *x, int x_et, int64_t ld_x, int m, uint8_t *codes,
                      uint8_t *scales, void *y, int et, int64_t ld) {
    const hipError_t e = mx4_quantize(L, x, nullptr, x_et, ld_x, m, k, nullptr, codes, scales);
    return e != hipSuccess ? e : mx4_gemm(L, w, ws, 1, rows, k, codes, scales, m, nullptr, nullptr, 0, 0, y, et, ld);
}

// ------------------------------------------------------------------------------------ a few tokens' experts

struct Mx4Moe {
    const uint8_t *wg, *wgs, *wu, *wus, *wd, *wds;
    u32 n_experts, hidden, ff, n_tokens, top_k;
    const void *x, *resid;
    size_t ld_x, ld_resid, ld_y;
    const u32 *sel;
    const float *w;
    float *h; // a row of ff values a slot
    void *y;
    GateRule rule;
    u32 *fault, layer;
};

// A row's share of lane `lane` of a dot with the values that `load` gives for eight of k at a time.
template <class F>
__device__ __forceinline__ float mx4_dot(const uint8_t *row, const uint8_t *scales, u32 k, u32 lane, F load) {
    float sum = 0.0f;
    for (u32 c = 8 * lane; c < k; c += 512) {
        float w[8], v[8];
        mx4_values(*reinterpret_cast<const u32 *>(row + c / 2), scales[c / 32], w);
        load(c, v);
#pragma unroll
        for (int j = 0; j < 8; j++) sum = fmaf(w[j], v[j], sum);
    }
    return wave_sum(sum);
}

// A wave a slot's value of h.
template <int ET>
__global__ __launch_bounds__(256) void k_mx4_moe_up(Mx4Moe a) {
    const u32 lane = threadIdx.x & 63, slot = blockIdx.y, f = blockIdx.x * 4 + (threadIdx.x >> 6), e = a.sel[slot];
    if (e >= a.n_experts) {
        if (e != 0xffffffffu && threadIdx.x == 0) bm_raise(a.fault, a.layer, kSiteExpertId);
        return;
    }
    if (f >= a.ff) return;
    const u32 kp = (a.hidden + 31) / 32 * 16, ks = (a.hidden + 511) / 512 * 16;
    const size_t row = (size_t)e * a.ff + f, x = (size_t)(slot / a.top_k) * a.ld_x;
    const auto load = [&](u32 c, float (&v)[8]) { elem_load_some<ET, 8>(a.x, x + c, a.hidden - c, v); };
    const float g = mx4_dot(a.wg + row * kp, a.wgs + row * ks, a.hidden, lane, load), u = mx4_dot(a.wu + row * kp, a.wus + row * ks, a.hidden, lane, load);
    if (lane) return;
    bool odd;
    a.h[(size_t)slot * a.ff + f] = bm_gate_rule(a.rule.act, a.rule.limit, g, u, odd);
    if (odd) bm_raise(a.fault, a.layer, kSiteF32Product);
}

// A wave a token's value of y.
template <int ET>
__global__ __launch_bounds__(256) void k_mx4_moe_down(Mx4Moe a) {
    const u32 lane = threadIdx.x & 63, token = blockIdx.y, r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= a.hidden) return;
    const u32 kp = (a.ff + 31) / 32 * 16, ks = (a.ff + 511) / 512 * 16;
    float sum = 0.0f;
    for (u32 s = token * a.top_k; s < (token + 1) * a.top_k; s++) {
        const u32 e = a.sel[s];
        if (e >= a.n_experts) continue;
        const size_t row = (size_t)e * a.hidden + r, h = (size_t)s * a.ff;
        sum = fmaf(a.w[s], mx4_dot(a.wd + row * kp, a.wds + row * ks, a.ff, lane, [&](u32 c, float (&v)[8]) { elem_load_some<kElemF32, 8>(a.h, h + c, a.ff - c, v); }), sum);
    }
    if (lane) return;
    if (a.resid) sum = __fadd_rn(sum, elem_load1<ET>(a.resid, token * a.ld_resid + r));
    elem_store1<ET>(a.y, token * a.ld_y + r, sum);
}

template <int ET>
static hipError_t moe_launch(const Launch &L, const Mx4Moe &a) {
    hipLaunchKernelGGL((k_mx4_moe_up<ET>), dim3((a.ff + 3) / 4, a.n_tokens * a.top_k), dim3(256), 0, L.stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_mx4_moe_down<ET>), dim3((a.hidden + 3) / 4, a.n_tokens), dim3(256), 0, L.stream, a);
    return hipGetLastError();
}

size_t mx4_moe_work(int n_tokens, int top_k, int, int ff) { return (size_t)n_tokens * top_k * ff * sizeof(float); }

hipError_t mx4_moe(const Launch &L, const Mx4Stack &g, const Mx4Stack &u, const Mx4Stack &d, int n_experts, int hidden, int ff, const void *x, int et,
                   int64_t ld_x, int n_tokens, const uint32_t *sel, const float *w, int top_k, const void *resid, int64_t ld_resid, void *y, int64_t ld_y,
                   void *work) {
    const Mx4Moe a = {g.w, g.scales, u.w, u.scales, d.w, d.scales, (u32)n_experts, (u32)hidden, (u32)ff, (u32)n_tokens, (u32)top_k, x, resid, (size_t)ld_x,
                      (size_t)ld_resid, (size_t)ld_y, sel, w, (float *)work, y, L.rule, L.fault, L.layer};
    if (et == kElemF32) return moe_launch<kElemF32>(L, a);
    if (et == kElemF16) return moe_launch<kElemF16>(L, a);
    return moe_launch<kElemBF16>(L, a);
}

} // namespace bmk
