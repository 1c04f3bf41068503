// The experts' product of rows and weights in 8-bit integers, each row and each output channel under a scale of its own (gfx950):
//
//   y[r, c] = act(s_r t_c sum_k q[r, k] w[c, k] + b[c])         gated: act(the same of Wg, bg) (the same of Wu, bu)
//
// The sums are 32-bit integers and exact; one rounding makes them float32, the scales, the bias and the activation are float32, one more rounding makes the
// result.  v_mfma_i32_16x16x64_i8 takes 16 bytes of a row per lane, as the 16-bit forms do, so slabs of 128 bytes, their LDS image and its swizzle are those of
// gemm_kernel.hpp.
//
// 128 x 128 tiles, four waves of 64 x 64 each, two slabs of LDS; two workgroups share a compute unit.  Gated: 64 columns of the gate and the same 64 of the linear half to
// a tile, 32 and 32 to a wave, so that a lane has both of its products.
#include "gemm_int8.hpp"
#include "gated_terms.hpp"

namespace fmoe {
namespace {
using namespace gemm;

typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int kThreadsI8 = 256, kTile = 128, kPart = kTile * kSlabBytes, kStage = 2 * kPart;

template <typename OUT, bool GATED>
__global__ __launch_bounds__(kThreadsI8, 2) void grouped_gemm_int8_kernel(const Int8Params prm) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only needs the launch stub
    constexpr uint32_t kOutOfRange = 0x80000000u;
    constexpr int kRsrcFlags = 0x00020000;   // raw buffer, 32-bit data format
    constexpr int kCols = GATED ? kTile / 2 : kTile;
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * kStage];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave >> 1, wn = wave & 1, lb = lane & 15, hq = lane >> 4;

    // which tile: a contiguous eighth of the logical order per XCD, kGroupM row tiles per column tile
    typedef const int32_t __attribute__((address_space(4))) *DevTab;    // read-only, uniform: scalar loads
    typedef const i32x4 __attribute__((address_space(4))) *DevTab4;
    const DevTab dtab = (DevTab)(uintptr_t)prm.dev_tab;
    const int tm_total = dtab[segtab::kTiles128], total = tm_total * prm.tiles_n, per_xcd = (total + 7) >> 3;
    const int L = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || L >= total) return;
    const int grp = L / (kGroupM * prm.tiles_n), in_grp = L - grp * kGroupM * prm.tiles_n, gsz = min(kGroupM, tm_total - grp * kGroupM);
    const int nt = in_grp / gsz, mt = grp * kGroupM + in_grp - nt * gsz;
    const i32x4 entry = *(DevTab4)(dtab + prm.map_off + 4 * mt);   // {expert, first row, rows}
    const int expert = entry[0], row0 = entry[1], q_valid = entry[2], n0 = nt * kCols, K = prm.k_extent;

    // memory -> LDS: thread t fetches, in pass it, the chunk that belongs in slot it * 256 + t: row it * 32 + t / 8, position t % 8
    uint32_t p_off[4], q_off[4];
    const int chunk = (t & 7) ^ swz((t >> 3) & 31);
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int r = it * 32 + (t >> 3);
        // gated: 32 columns of the gate and 32 of the linear half to each half of the tile's rows of w
        const int col = n0 + (GATED ? (it >> 1) * 32 + (t >> 3) : r), w_row = col + (GATED && (it & 1) ? prm.n_cols : 0);
        p_off[it] = col < prm.n_cols ? (uint32_t)(w_row * (int)prm.ldw + chunk * 16) : kOutOfRange;
        q_off[it] = r < q_valid ? (uint32_t)(r * (int)prm.ldx + chunk * 16) : kOutOfRange;
    }
    auto resource = [&](const int8_t *p) {
        const uint64_t a = (uint64_t)p;
        i32x4 rs;
        rs[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
        rs[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu));
        rs[2] = (int)kOutOfRange;
        rs[3] = kRsrcFlags;
        return rs;
    };
    const i32x4 p_rs = resource(prm.w + (int64_t)expert * prm.w_expert_stride), q_rs = resource(prm.x + (int64_t)row0 * prm.ldx);
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)smem;
    auto issue = [&](int k0, int buf) {
        const uint32_t past = (uint32_t)(K - 1 - k0 - chunk * 16) & kOutOfRange;   // the chunk begins past the contraction
        const int from = __builtin_amdgcn_readfirstlane(k0);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const uint32_t at = __builtin_amdgcn_readfirstlane(lds_base + buf * kStage + part * kPart + it * 4096 + wave * 1024);
                asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                             :
                             : "s"(at), "v"((part ? q_off[it] : p_off[it]) | past), "s"(part ? q_rs : p_rs), "s"(from)
                             : "memory", "m0");
            }
    };
    i32x4 acc[4][4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = i32x4{0, 0, 0, 0};
    const int n_slabs = (K + kSlabBytes - 1) / kSlabBytes;
    issue(0, 0);
    for (int s = 0; s < n_slabs; ++s) {
        __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1 < n_slabs) issue((s + 1) * kSlabBytes, (s + 1) & 1);
        const unsigned char *sp = smem + (s & 1) * kStage, *sq = sp + kPart;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            i32x4 pf[4], qf[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int pr = 64 * wn + 16 * x + lb, qr = 64 * wm + 16 * x + lb;
                pf[x] = *(const i32x4 *)(sp + pr * kSlabBytes + (((4 * ks + hq) ^ swz(pr)) << 4));
                qf[x] = *(const i32x4 *)(sq + qr * kSlabBytes + (((4 * ks + hq) ^ swz(qr)) << 4));
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pf[x], qf[y], acc[x][y], 0, 0, 0);
        }
    }
    // acc[x][y][i] is row 64 wm + 16 y + lb, row 64 wn + 16 x + 4 hq + i of the tile's weights
    constexpr int kBlocks = GATED ? 2 : 4;
    const int64_t w_rows = (int64_t)prm.n_cols * (GATED ? 2 : 1);
    const float *t_c = prm.w_scale + expert * w_rows;
    const OUT *bias = prm.bias ? (const OUT *)prm.bias + expert * w_rows : nullptr;
    const bool whole = (prm.n_cols & 3) == 0;
#pragma unroll
    for (int x = 0; x < kBlocks; ++x) {
        const int col = n0 + (GATED ? 32 : 64) * wn + 16 * x + 4 * hq;
        float scale[GATED ? 2 : 1][4], add[GATED ? 2 : 1][4];
#pragma unroll
        for (int half = 0; half < (GATED ? 2 : 1); ++half)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = col + i < prm.n_cols;
                const int64_t c = (int64_t)half * prm.n_cols + col + i;
                scale[half][i] = in ? t_c[c] : 0.f;
                add[half][i] = in && bias ? (float)bias[c] : 0.f;
            }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int r = 64 * wm + 16 * y + lb;
            if (r >= q_valid || col >= prm.n_cols) continue;
            const float s = prm.x_scale[row0 + r];
            struct alignas(4 * sizeof(OUT)) Four { OUT v[4]; } out;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float g = fmaf((float)acc[x][y][i], s * scale[0][i], add[0][i]);
                float v = gate_act<sizeof(OUT) == 2>(g, prm.activation);
                if constexpr (GATED) v *= fmaf((float)acc[x + 2][y][i], s * scale[1][i], add[1][i]);
                out.v[i] = (OUT)v;
            }
            OUT *at = (OUT *)prm.y + (int64_t)(row0 + r) * prm.n_cols + col;
            if (whole) {
                *(Four *)at = out;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < prm.n_cols) at[i] = out.v[i];
            }
        }
    }
#endif
}

template <typename OUT> int launch(Int8Params prm, hipStream_t stream) {
    prm.tiles_n = (int)ceil_div(prm.n_cols, prm.gated ? kTile / 2 : kTile);
    prm.map_off = (int)segtab::map128_off(prm.rows_cap, prm.n_expert);
    const int64_t grid = ceil_div(segtab::cap_tiles(prm.rows_cap, prm.n_expert, kTile) * prm.tiles_n, 8) * 8;
    if (grid > kMostThreads / kThreadsI8 || grid > (int64_t)INT32_MAX) return fail(FMOE_ELIMIT, "int8 product: grid of %lld workgroups", (long long)grid);
    if (prm.gated) grouped_gemm_int8_kernel<OUT, true><<<(unsigned)grid, kThreadsI8, 0, stream>>>(prm);
    else grouped_gemm_int8_kernel<OUT, false><<<(unsigned)grid, kThreadsI8, 0, stream>>>(prm);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_linear_int8(const void *x, int64_t ldx, const void *x_scale, const void *w, int64_t ldw, int64_t w_expert_stride,
                                const void *w_scale, const void *bias, void *y, const void *segment_table, int64_t n_expert, int64_t rows_cap,
                                int64_t in_feat, int64_t out_feat, int gated, int activation, int dtype, void *workspace, int64_t workspace_bytes,
                                void *stream) {
    const char *who = "fmoe_linear_int8";
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who, dtype);
    FMOE_REQUIRE(is_gate_activation(activation), "%s: unknown activation %d", who, activation);
    FMOE_REQUIRE(n_expert >= 1 && rows_cap >= 0 && in_feat >= 1 && out_feat >= 1, "%s: bad sizes", who);
    const int64_t whole = ceil_div(in_feat, 16) * 16, w_rows = out_feat * (gated ? 2 : 1);
    // (131072 products of numbers up to 128: below 2^31)
    if (in_feat > 131072 || n_expert > (1 << 24) || rows_cap > (int64_t)INT32_MAX - 65536 || out_feat > (1 << 28) || ldx > (1 << 22) ||
        ldw > (1 << 28) || w_rows * ldw >= ((int64_t)1 << 31))
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    FMOE_REQUIRE(ldx >= whole && ldw >= whole && ldx % 16 == 0 && ldw % 16 == 0 && w_expert_stride % 16 == 0 && w_expert_stride >= 0,
                 "%s: rows of 8-bit integers begin on 16 bytes, at least %lld apart", who, (long long)whole);
    if (rows_cap == 0) return FMOE_OK;
    FMOE_REQUIRE(x && x_scale && w && w_scale && y && segment_table, "%s: NULL pointer", who);
    FMOE_REQUIRE(aligned16(x) && aligned16(w) && aligned16(segment_table) && (reinterpret_cast<uintptr_t>(y) & 15) == 0, "%s: tensors begin on 16 bytes", who);
    Int8Params prm{};
    prm.x = (const int8_t *)x; prm.w = (const int8_t *)w; prm.x_scale = (const float *)x_scale; prm.w_scale = (const float *)w_scale;
    prm.bias = bias; prm.y = y; prm.ldx = ldx; prm.ldw = ldw; prm.w_expert_stride = w_expert_stride;
    prm.n_cols = (int)out_feat; prm.k_extent = (int)whole; prm.gated = gated != 0; prm.activation = activation;
    prm.dev_tab = (const int32_t *)segment_table; prm.n_expert = n_expert; prm.rows_cap = rows_cap; prm.dtype = dtype;
    if (int8_in_pairs(prm)) return launch_int8_pairs(prm, workspace, workspace_bytes, (hipStream_t)stream);
    if (dtype == FMOE_F32) return launch<float>(prm, (hipStream_t)stream);
    return dtype == FMOE_BF16 ? launch<__bf16>(prm, (hipStream_t)stream) : launch<_Float16>(prm, (hipStream_t)stream);
}

extern "C" int64_t fmoe_linear_int8_workspace_bytes(int64_t n_expert, int64_t rows_cap, int64_t in_feat, int64_t out_feat, int gated, int dtype) {
    if (n_expert < 1 || rows_cap < 1 || in_feat < 1 || in_feat > 131072 || out_feat < 1 || out_feat > (1 << 28)) return 0;
    Int8Params prm{};
    prm.n_expert = n_expert; prm.rows_cap = rows_cap; prm.n_cols = (int)out_feat; prm.k_extent = (int)(ceil_div(in_feat, 16) * 16);
    prm.gated = gated != 0; prm.dtype = dtype;
    return int8_in_pairs(prm) ? int8_workspace_bytes(prm) : 0;
}
