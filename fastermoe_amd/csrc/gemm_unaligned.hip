// Grouped GEMM over ragged expert segments for 16-bit types whose feature sizes or pointers are off the
// 16-byte grid (gfx950), on the 16 x 16 x 32 MFMA.
//
// The aligned kernels bring slabs straight from memory into LDS, which needs 16-byte chunks on 16-byte boundaries.
// Here a chunk of eight elements comes in through registers with one 16-byte load from wherever it begins (global
// loads take any alignment) and goes to the same LDS image as in gemm_kernel.hpp, so that the fragment reads
// and products are the same.  Where the contraction or the row of a [contraction][index] operand ends inside a chunk, the
// chunk that ends with it is read and moved down; rows past a tile's end repeat its last row and are not stored.
//
// 128 x 128 tiles (64 x 64 per wave), 64 x 128 where those would leave compute units without one; the next slab's chunks are requested before the products of the current
// one.  Forward products and data gradients have one slab of LDS, so that registers alone decide how many workgroups share a compute unit, and one computes while others
// wait: four with 64-row forward products, three with 64-row data gradients and 128-row gated forwards, two with the other 128-row tiles.  Weight gradients, two to a
// unit either way, have two slabs and a barrier less.  us of the kernel with one / two slabs, bfloat16: gated forward, 8192 rows, 8 experts of 1023 -> 2 x 2047: 127 / 148, of
// 2047 -> 2 x 4093: 520 / 584, 32768 rows, 8 of 1022 -> 2 x 4090: 922 / 1006; plain, 16384 rows, 16 of 1001 x 1003: 82 / 84, with an activation 103 / 101; data gradients, 8192 rows, 8
// of 2047 x 4093: 317 / 324 (within 1 % on average); weight gradients there 302 / 299, 8 of 1023 x 2047: 83 / 79, 1554 rows, 12 of 500 x 2604: 27.7 / 26.5.
// Bound by the latency of those
// loads up to a few hundred rows per expert (1.2 us a slab) and by their way through registers above (600 TFLOP/s there).  Where few tiles have long contractions, a gated block's products share them between workgroups (launch_parts; see unaligned_parts() in
// grouped_gemm.hip).  The epilogues of gated products are those of gemm_kernel.hpp: 1554 rows, 12 experts of 500 -> 2 x 1302 in float16, 26 us forward and 22 for the
// gradient.  Measured against the element-wise kernel it replaced: see the dispatch in grouped_gemm.hip.
#include "gemm_kernel.hpp"
#include "unaligned_loads.hpp"

#include <optional>

namespace fmoe {
namespace {
using namespace gemm;

// the first n floats (4 or more: four) of four from or to wherever they begin
__device__ __forceinline__ f32x4 load_floats(const float *p, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        __builtin_memcpy(&v, p, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < n) v[j] = p[j];
    }
    return v;
}
__device__ __forceinline__ void store_floats(float *p, const f32x4 &v, int n) {
    if (n >= 4) {
        __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < n) p[j] = v[j];
    }
}

constexpr int kUaThreads = 256, kUaBN = 128, kUaBK = 64;

// the float32 sums of a part of the contraction instead of an epilogue: see launch_parts
constexpr int kEpiParts = 100;
__host__ __device__ __forceinline__ int parts_ld(int n_cols) { return (n_cols + 3) & ~3; }   // floats from row to row of those

// Slabs of LDS: see above
constexpr int slabs_of(int ragged) { return ragged == kRaggedK ? 2 : 1; }

// PSHAPE / QSHAPE: kKC = [index][contraction] in memory, kMC = [contraction][index].  EPI: kEpiGated, kEpiDGated, kEpiParts, or 0: what the parameters say.
template <typename T, int BM, int PSHAPE, int QSHAPE, int RAGGED, int EPI>
__global__ __launch_bounds__(kUaThreads) void grouped_gemm_unaligned_kernel(const GemmParams prm) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only needs the launch stub
    static_assert(QSHAPE == kKC || BM == 128, "the swizzle of a [contraction][index] slab needs rows of 256 bytes");
    constexpr int BN = kUaBN, BK = kUaBK, TI = 4, TJ = BM / 32;
    constexpr int NP = BN * 8 / kUaThreads, NQ = BM * 8 / kUaThreads;   // chunks per thread and slab
    constexpr int P_BYTES = BN * 128, Q_BYTES = BM * 128, STAGE = P_BYTES + Q_BYTES;
    constexpr bool kBiasGrad = RAGGED == kRaggedK;
    constexpr bool kHalves = epi_halves(EPI);
    constexpr int kCols = kHalves ? BN / 2 : BN;   // C columns of a tile
    constexpr int kSlabs = slabs_of(RAGGED);
    __shared__ __attribute__((aligned(16))) unsigned char smem[kSlabs * STAGE];

    if constexpr (EPI == kEpiGated || EPI == kEpiDGated) {
        const int64_t there = ((const int32_t __attribute__((address_space(4))) *)(uintptr_t)prm.dev_tab)[segtab::kRows];
        if (prm.tail != nullptr && there < prm.tail_rows)
            for (int64_t i = (int64_t)blockIdx.x * kUaThreads + threadIdx.x; i < (prm.tail_rows - there) * prm.tail_elems; i += (int64_t)gridDim.x * kUaThreads)
                ((T *)prm.tail)[there * prm.tail_elems + i] = (T)0.f;
    }

    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave >> 1, wn = wave & 1, lb = lane & 15, hq = lane >> 4;

    // -- which tile: a contiguous eighth of the logical order per XCD, kGroupM row tiles per column tile
    // (over a device table the launch is sized for the most tiles there can be)
    typedef const int32_t __attribute__((address_space(4))) *DevTab;    // read-only, uniform: scalar loads
    const DevTab dtab = (DevTab)(uintptr_t)prm.dev_tab;
    const bool dev = prm.dev_tab != nullptr;
    int tm_total = prm.tiles_m, total_tiles = prm.total_tiles;
    if (RAGGED == kRaggedRows) {
        tm_total = dev ? dtab[segtab::kTiles128] * (128 / BM) : prm.tab.tile[prm.tab.n];
        total_tiles = tm_total * prm.tiles_n * (EPI == kEpiParts ? prm.k_split : 1);
    }
    const int per_xcd = (total_tiles + 7) >> 3;
    const int L = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || L >= total_tiles) return;
    int ei = 0, rem = L;
    if (RAGGED == kRaggedK) {
        ei = L / (prm.tiles_m * prm.tiles_n);
        rem = L - ei * (prm.tiles_m * prm.tiles_n);
    }
    const int part = EPI == kEpiParts ? rem % prm.k_split : 0;
    if (EPI == kEpiParts) rem /= prm.k_split;
    const int grp = rem / (kGroupM * prm.tiles_n), in_grp = rem - grp * kGroupM * prm.tiles_n;
    const int gsz = min(kGroupM, tm_total - grp * kGroupM);
    const int nt = in_grp / gsz, mt = grp * kGroupM + in_grp - nt * gsz;
    int seg_lo, seg_hi, row0 = 0;   // (ragged rows over a device table: of this very tile)
    if (RAGGED == kRaggedRows && dev) {
        typedef int i32x4 __attribute__((ext_vector_type(4)));
        typedef const i32x4 __attribute__((address_space(4))) *DevTab4;
        constexpr int kPerEntry = 128 / BM;   // (tiles of 64 rows: the halves of the map's 128; the second may have no rows)
        const i32x4 entry = *(DevTab4)(dtab + prm.dev_map_off + 4 * (mt / kPerEntry));
        ei = entry[0];
        seg_hi = entry[1] + entry[2];
        row0 = seg_lo = entry[1] + (mt % kPerEntry) * BM;
        if (seg_lo >= seg_hi) return;
    } else if (RAGGED == kRaggedRows) {
        int lo = 0, hi = prm.tab.n;  // tile[lo] <= mt < tile[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prm.tab.tile[mid] <= mt) lo = mid; else hi = mid;
        }
        ei = lo;
        seg_lo = prm.tab.seg[ei];
        seg_hi = prm.tab.seg[ei + 1];
        row0 = seg_lo + (mt - prm.tab.tile[ei]) * BM;
    } else {
        seg_lo = dev ? dtab[segtab::kHeader + ei] : prm.tab.seg[ei];
        seg_hi = dev ? dtab[segtab::kHeader + ei + 1] : prm.tab.seg[ei + 1];
    }
    const int expert = prm.tab.first_expert + ei;
    const int n0 = nt * kCols, p_valid = min(kCols, prm.n_cols - n0);
    int K, q_valid, m0 = 0;
    const T *P, *Q;
    int64_t c_off;
    if (RAGGED == kRaggedRows) {
        q_valid = min(BM, seg_hi - row0);
        K = prm.k_extent;
        P = (const T *)prm.P + (int64_t)expert * prm.p_expert_stride + (PSHAPE == kKC ? (int64_t)n0 * prm.ldp : (int64_t)n0);
        Q = (const T *)prm.Q + (int64_t)row0 * prm.ldq;
        c_off = (int64_t)row0 * prm.ldc + n0;
        if (EPI == kEpiParts) {
            const int k_lo = part * prm.split_slabs * BK;
            P += PSHAPE == kKC ? (int64_t)k_lo : (int64_t)k_lo * prm.ldp;
            Q += k_lo;
            K = min(K - k_lo, prm.split_slabs * BK);   // (no part is empty)
        }
    } else {
        m0 = mt * BM;
        q_valid = min(BM, prm.n_rows - m0);
        K = seg_hi - seg_lo;
        P = (const T *)prm.P + (int64_t)seg_lo * prm.ldp + n0;
        Q = (const T *)prm.Q + (int64_t)seg_lo * prm.ldq + m0;
        c_off = (int64_t)expert * prm.c_expert_stride + (int64_t)m0 * prm.ldc + n0;
    }

    // An expert without rows: its tiles write zeros over equal parts of its gradient, which is dense (as a tile of no
    // slabs, stored 16 bytes at a time off the grid: 1 row over 500 experts of 1483 x 70, 91 us, like this 23).
    if (RAGGED == kRaggedK && K == 0 && !(prm.accumulate_first && ei == 0)) {
        const int64_t size = (int64_t)prm.n_rows * prm.n_cols, per = (size + prm.tiles_m * prm.tiles_n - 1) / (prm.tiles_m * prm.tiles_n);
        const int64_t lo = min(rem * per, size), hi = min(lo + per, size);
        T *gw = (T *)prm.C + (int64_t)expert * prm.c_expert_stride;
        const int64_t body = min(lo + (int64_t)((16 - ((uintptr_t)(gw + lo) & 15)) & 15) / 2, hi), vecs = (hi - body) / 8;
        for (int64_t i = lo + t; i < body; i += kUaThreads) gw[i] = (T)0.f;
        for (int64_t v = t; v < vecs; v += kUaThreads) ((u32x4 *)(gw + body))[v] = u32x4{0u, 0u, 0u, 0u};
        for (int64_t i = body + 8 * vecs + t; i < hi; i += kUaThreads) gw[i] = (T)0.f;
        if (rem == 0 && prm.bias_grad != nullptr)
            for (int r = t; r < prm.n_rows; r += kUaThreads) ((T *)prm.bias_grad)[(int64_t)expert * prm.n_rows + r] = (T)0.f;
        return;
    }

    // -- memory -> registers -> LDS: thread t has chunk it * 256 + t of the slab
    auto chunk_index = [&](int shape, int it) { return shape == kKC ? (it * kUaThreads + t) >> 3 : (it * kUaThreads + t) >> 4; };
    // (its offsets from the slab's first element do not change: rows and chunks past a tile's end repeat the last one)
    int64_t p_off[NP], q_off[NQ];
    auto set_offsets = [&](int shape, int64_t *off, int n, int64_t ld, int valid) {
#pragma unroll
        for (int it = 0; it < n; ++it) {
            const int r = chunk_index(shape, it);
            off[it] = shape == kKC ? (int64_t)min(r, valid - 1) * ld + (t & 7) * 8 : (int64_t)r * ld + min((t & 15) * 8, (valid - 1) & ~7);
        }
    };
    set_offsets(PSHAPE, p_off, NP, prm.ldp, p_valid);
    if constexpr (kHalves) {
        // 32 rows of the gate's weights, the same 32 of the linear half's, to each pair of waves
#pragma unroll
        for (int it = 0; it < NP; ++it) {
            const int r = chunk_index(kKC, it), col = (r >> 6) * 32 + (r & 31);
            p_off[it] = ((int64_t)min(col, p_valid - 1) + ((r >> 5) & 1 ? prm.n_cols : 0)) * prm.ldp + (t & 7) * 8;
        }
    }
    set_offsets(QSHAPE, q_off, NQ, prm.ldq, q_valid);
    auto fetch = [&](int shape, u32x4 *dst, int n, const T *base, const int64_t *off, int64_t ld, int valid, int extent,
                     int row_elems, int k0) {
        const T *slab = base + (shape == kKC ? (int64_t)k0 : (int64_t)k0 * ld);
        // A chunk that runs past the end of its [contraction][index] row brings in what is not stored: the first
        // elements of the row below, of which there is one unless this is the last slab.  (Nothing touches what these
        // loads return before the products of the slab before; the other branch waits for its loads at once.)
        if (k0 + BK <= K && (shape == kKC || valid == extent || (k0 + BK < K && row_elems >= 8))) {
#pragma unroll
            for (int it = 0; it < n; ++it) dst[it] = load_unaligned(slab + off[it]);
        } else {
            const bool back = (shape == kKC ? K : row_elems) >= 8;
            const T *safe = shape == kKC ? base : base + min(0, valid - 8);
#pragma unroll
            for (int it = 0; it < n; ++it) {
                const int r = chunk_index(shape, it);
                const int left = shape == kKC ? K - k0 - (t & 7) * 8 : (k0 + r < K ? valid - min((t & 15) * 8, (valid - 1) & ~7) : 0);
                dst[it] = load_part(slab + off[it], safe, left, back);
            }
        }
    };
    auto put = [&](int shape, const u32x4 *src, int n, unsigned char *to) {
        for (int it = 0; it < n; ++it) {
            const int r = chunk_index(shape, it);
            const int at = shape == kKC ? r * 128 + (((t & 7) ^ swz(r)) << 4) : r * 256 + (((t & 15) ^ mc_swz<T>(r)) << 4);
            *(u32x4 *)(to + at) = src[it];
        }
    };
    // -- fragments, as in gemm_kernel.hpp: block j of step ks
    auto frag = [&](int shape, const unsigned char *buf, int j, int ks) -> u32x4 {
        if (shape == kKC) return *(const u32x4 *)(buf + (16 * j + lb) * 128 + (((4 * ks + hq) ^ swz(lb)) << 4));
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_ptr;
        const int kb = ks * 32 + hq * 8 + (lb >> 2);
        const unsigned char *at = buf + kb * 256 + (((2 * j + ((lb >> 1) & 1)) ^ mc_swz<T>(kb)) << 4) + (lb & 1) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + 1024));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        return u32x4{l2[0], l2[1], h2[0], h2[1]};
    };

    // a barrier for what lies in LDS (loads into registers go on)
    auto lds_barrier = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    // Block row y of a wave.  Ragged rows: every other one, so that both pairs of waves have some of an expert's few
    // rows and the epilogue ends at the last of them.
    auto row_block = [&](int y) { return RAGGED == kRaggedRows ? 2 * y + wm : TJ * wm + y; };

    f32x4 acc[TI][TJ], bacc[kBiasGrad ? TJ : 1];
#pragma unroll
    for (int x = 0; x < TI; ++x)
#pragma unroll
        for (int y = 0; y < TJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (kBiasGrad) {
#pragma unroll
        for (int y = 0; y < TJ; ++y) bacc[y] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const bool want_bias = kBiasGrad && prm.bias_grad != nullptr && n0 == 0 && wn == 0;
    const uint32_t one2 = std::is_same<T, __bf16>::value ? 0x3f803f80u : 0x3c003c00u;
    const u32x4 ones = {one2, one2, one2, one2};

    u32x4 pr[NP], qr[NQ];
    const int n_slabs = (K + BK - 1) / BK;
    if (n_slabs > 0) {
        fetch(PSHAPE, pr, NP, P, p_off, prm.ldp, p_valid, BN, prm.n_cols, 0);
        fetch(QSHAPE, qr, NQ, Q, q_off, prm.ldq, q_valid, BM, prm.n_rows, 0);
    }
    for (int s = 0; s < n_slabs; ++s) {
        unsigned char *buf = smem + (kSlabs == 2 ? s & 1 : 0) * STAGE;
        if (kSlabs == 1 && s > 0) lds_barrier();   // (the slab before has been read; with two: the one before that, ahead of the last barrier)
        put(PSHAPE, pr, NP, buf);
        put(QSHAPE, qr, NQ, buf + P_BYTES);
        lds_barrier();
        if (s + 1 < n_slabs) {
            fetch(PSHAPE, pr, NP, P, p_off, prm.ldp, p_valid, BN, prm.n_cols, (s + 1) * BK);
            fetch(QSHAPE, qr, NQ, Q, q_off, prm.ldq, q_valid, BM, prm.n_rows, (s + 1) * BK);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            u32x4 pf[TI], qf[TJ];
#pragma unroll
            for (int x = 0; x < TI; ++x) pf[x] = frag(PSHAPE, buf, wn * TI + x, ks);
#pragma unroll
            for (int y = 0; y < TJ; ++y) qf[y] = frag(QSHAPE, buf + P_BYTES, row_block(y), ks);
#pragma unroll
            for (int x = 0; x < TI; ++x)
#pragma unroll
                for (int y = 0; y < TJ; ++y) Elem<T>::mma(acc[x][y], pf[x], qf[y]);
            if (kBiasGrad && want_bias) {
#pragma unroll
                for (int y = 0; y < TJ; ++y) Elem<T>::mma(bacc[y], ones, qf[y]);
            }
        }
    }
    __syncthreads();

    auto wave_sync = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    if constexpr (EPI == kEpiParts) {
        const int ld = parts_ld(prm.n_cols);
        float *to = prm.split_ws + ((int64_t)part * prm.dev_rows_cap + row0) * ld + n0;
#pragma unroll
        for (int y = 0; y < TJ; ++y) {
            const int row = 16 * row_block(y) + lb;
            if (row >= q_valid) continue;
#pragma unroll
            for (int x = 0; x < TI; ++x) {
                const int col = 64 * wn + 16 * x + 4 * hq;
                if (col < p_valid) *(f32x4 *)(to + (int64_t)row * ld + col) = acc[x][y];
            }
        }
        return;
    }
    if constexpr (EPI == kEpiGated || EPI == kEpiDGated) {
        // Gated products: sixteen rows at a time, 64 columns of C (dg and du), or 32 of each half, through 2 KiB of LDS per wave and matrix
        constexpr int kWaveCols = kHalves ? 32 : 64, kPieces = kWaveCols / 8, kSteps = kPieces / 4, kRows = 64 / kPieces;
        unsigned char *area = smem + wave * 4096;
        const int io_r = lane / kPieces, io_c = lane % kPieces, wave_col = kWaveCols * wn;
        auto at4 = [&](int a, int x) { return (u32x2 *)(area + a * 2048 + lb * (kPieces * 16) + (((2 * x + (hq >> 1)) ^ (lb & (kPieces - 1))) << 4) + (hq & 1) * 8); };
        auto piece = [&](int a, int i) {
            const int r = i * kRows + io_r;
            return (u32x4 *)(area + a * 2048 + r * (kPieces * 16) + ((io_c ^ (r & (kPieces - 1))) << 4));
        };
        // this lane's eight elements of step i of block row y: row in the tile, columns left of its eight (0 or less: none)
        auto row_of = [&](int y, int i) { return 16 * row_block(y) + i * kRows + io_r; };
        const int left = p_valid - (wave_col + io_c * 8);
        auto store = [&](int a, T *to, int64_t ld, int y) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (row_of(y, i) < q_valid && left > 0) store_some(to + (int64_t)row_of(y, i) * ld + wave_col + io_c * 8, *piece(a, i), left);
        };
        if constexpr (kHalves) {
            const T *bias = prm.bias ? (const T *)prm.bias + (int64_t)expert * prm.bias_expert_stride + n0 : nullptr;
            float bias_of[TI][4];
#pragma unroll
            for (int x = 0; x < TI; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = wave_col + 16 * (x & 1) + 4 * hq + i;
                    bias_of[x][i] = bias != nullptr && col < p_valid ? (float)bias[col + (x < 2 ? 0 : prm.n_cols)] : 0.f;
                }
            float *pre = prm.aux ? (float *)prm.aux + 2 * c_off - n0 : nullptr;
#pragma unroll
            for (int y = 0; y < TJ; ++y) {
                if (16 * row_block(y) >= q_valid) break;
                // float32, from the lanes that hold them (through LDS, 128 bytes of a row at a time: 8192 rows, 8 experts of 2047 -> 2 x 4093, 910 us both products, 840 so)
                if (pre != nullptr) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            f32x4 v = acc[x + 2 * h][y];
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] += bias_of[x + 2 * h][i];
                            const int row = 16 * row_block(y) + lb, c = wave_col + 16 * x + 4 * hq;
                            if (row < q_valid && c < p_valid) store_floats(pre + (int64_t)row * (2 * prm.ldc) + c + (h ? prm.n_cols : 0), v, p_valid - c);
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    alignas(8) T v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float g = acc[x][y][i] + bias_of[x][i], u = acc[x + 2][y][i] + bias_of[x + 2][i];
                        v[i] = (T)(gate_act<true>(g, prm.activation) * u);
                    }
                    *at4(0, x) = *(const u32x2 *)v;
                }
                wave_sync();
                store(0, (T *)prm.C + c_off, prm.ldc, y);
                wave_sync();
            }
        } else {
            // g and u (float32) straight to the lanes that hold their columns' sums
            const float *in = (const float *)prm.aux + c_off;
            T *out = (T *)prm.C + c_off;
#pragma unroll
            for (int y = 0; y < TJ; ++y) {
                if (16 * row_block(y) >= q_valid) break;
                const int row = 16 * row_block(y) + lb;
                f32x4 held[2][TI];
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int x = 0; x < TI; ++x) {
                        const int c = wave_col + 16 * x + 4 * hq;
                        held[a][x] = row < q_valid && c < p_valid ? load_floats(in + (int64_t)row * prm.ldc + c + a * prm.n_cols, p_valid - c) : f32x4{0.f, 0.f, 0.f, 0.f};
                    }
#pragma unroll
                for (int x = 0; x < TI; ++x) {
                    alignas(8) T g[4], u[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const ActTerms terms = gate_terms<true>(held[0][x][i], prm.activation);
                        const float dm = acc[x][y][i];
                        g[i] = (T)(dm * held[1][x][i] * terms.slope);
                        u[i] = (T)(dm * terms.value);
                    }
                    *at4(0, x) = *(const u32x2 *)g;
                    *at4(1, x) = *(const u32x2 *)u;
                }
                wave_sync();
                store(0, out, prm.ldc, y);
                store(1, out + prm.n_cols, prm.ldc, y);
                wave_sync();
            }
        }
        return;
    }
    // -- epilogue: acc[x][y][i] is C(row 16 row_block(y) + lb, column 64 wn + 16 x + 4 hq + i); sixteen rows at a
    // time through 2 KiB of LDS per wave and out as 128-byte row pieces
    unsigned char *stg = smem + wave * 2048;
    T *C = (T *)prm.C + c_off, *aux = prm.aux ? (T *)prm.aux + c_off : nullptr;
    const bool accumulate = RAGGED == kRaggedK && prm.accumulate_first && ei == 0;
    const T *bias = prm.bias ? (const T *)prm.bias + (int64_t)expert * prm.bias_expert_stride + n0 : nullptr;
    // (read once: in the loop, behind stores that might reach it as far as the compiler can tell, every use waited for those.  Forward
    // with GELU, 8192 rows, 8 experts of 2047 x 4093: 275 -> 225 us; with the epilogue's end at an expert's last rows
    // 556 rows, 64 of 38 x 1990: 50 -> 23)
    float bias_of[TI][4];
#pragma unroll
    for (int x = 0; x < TI; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 64 * wn + 16 * x + 4 * hq + i;
            bias_of[x][i] = bias != nullptr && col < p_valid ? (float)bias[col] : 0.f;
        }
    auto store_rows = [&](T *to, int y) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = i * 8 + (lane >> 3), c = lane & 7;
            const u32x4 v = *(const u32x4 *)(stg + r * 128 + ((c ^ (r & 7)) << 4));
            const int row = 16 * row_block(y) + r, col = 64 * wn + c * 8;
            if (row < q_valid && col < p_valid) {
                T *p = to + (int64_t)row * prm.ldc + col;
                if (col + 8 <= p_valid) {
                    __builtin_memcpy(p, &v, 16);
                } else {
                    const T *e = (const T *)&v;
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (col + j < p_valid) p[j] = e[j];
                }
            }
        }
        wave_sync();
    };
#pragma unroll
    for (int y = 0; y < TJ; ++y) {
        if (16 * row_block(y) >= q_valid) break;
        const int row = 16 * row_block(y) + lb;
#pragma unroll
        for (int kind = 1; kind >= 0; --kind) {   // 1: the pre-activation, 0: the result
            if (kind == 1 && (prm.epilogue != kEpiBiasAct || aux == nullptr)) continue;
#pragma unroll
            for (int x = 0; x < TI; ++x) {
                alignas(8) T res[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = 64 * wn + 16 * x + 4 * hq + i;
                    const bool in = row < q_valid && col < p_valid;
                    float v = acc[x][y][i] + bias_of[x][i];
                    if (kind == 0 && prm.epilogue == kEpiBiasAct) v = apply_act<false>(v, prm.activation);
                    if (prm.epilogue == kEpiDAct) v *= act_grad<false>(in ? (float)aux[(int64_t)row * prm.ldc + col] : 0.f, prm.activation);
                    if (accumulate) v += in ? (float)C[(int64_t)row * prm.ldc + col] : 0.f;
                    res[i] = (T)v;
                }
                *(u32x2 *)(stg + lb * 128 + (((2 * x + (hq >> 1)) ^ (lb & 7)) << 4) + (hq & 1) * 8) = *(const u32x2 *)res;
            }
            store_rows(kind == 1 ? aux : C, y);
        }
        if (kBiasGrad && want_bias && hq == 0 && row < q_valid) {
            T *dst = (T *)prm.bias_grad + (int64_t)expert * prm.n_rows + m0 + row;
            *dst = (T)(bacc[y][0] + (accumulate ? (float)*dst : 0.f));
        }
    }
#endif
}

// The parts' sums in ascending order, with the bias, in the results' type: sixteen rows of a tile of the table's and 256 columns to a workgroup, four columns to a lane.
template <typename T> __global__ __launch_bounds__(kUaThreads) void add_parts_kernel(const GemmParams prm) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const int32_t *dtab = prm.dev_tab;
    const int place = blockIdx.x >> 3;
    if (place >= dtab[segtab::kTiles128]) return;
    const i32x4 entry = *(const i32x4 *)(dtab + prm.dev_map_off + 4 * place);   // {expert, first row, rows}
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.y * 256 + lane * 4, ld = parts_ld(prm.n_cols);
    if (col >= prm.n_cols) return;
    const int n = min(4, prm.n_cols - col);
    float b[4] = {};
    if (prm.bias != nullptr)
        for (int i = 0; i < n; ++i) b[i] = (float)((const T *)prm.bias)[(int64_t)entry[0] * prm.bias_expert_stride + col + i];
    const int in_tile = (blockIdx.x & 7) * 16 + wave * 4;
    const int64_t row = entry[1] + in_tile;
    // (four rows of two parts on their way at a time)
    f32x4 sum[4] = {};
    for (int p = 0; p < prm.k_split; p += 2) {
        f32x4 v[2][4] = {};
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p + q < prm.k_split && in_tile + j < entry[2])
                    v[q][j] = *(const f32x4 *)(prm.split_ws + ((int64_t)(p + q) * prm.dev_rows_cap + row + j) * ld + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = (sum[j] + v[0][j]) + v[1][j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (in_tile + j >= entry[2]) return;
        T *to = (T *)prm.C + (row + j) * prm.ldc + col;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) to[i] = (T)(sum[j][i] + b[i]);
    }
#endif
}

template <typename T, int BM, int PS, int QS, int RG, int EPI = 0>
int launch_unaligned_tiles(GemmParams &prm, int epilogue, hipStream_t stream) {
    prm.epilogue = epilogue;
    prm.tiles_n = (int)ceil_div(prm.n_cols, epi_halves(EPI) ? kUaBN / 2 : kUaBN);
    prm.tiles_m = RG == kRaggedRows ? 0 : (int)ceil_div(prm.n_rows, BM);
    int64_t row_tiles = (int64_t)prm.tab.n * prm.tiles_m;
    if (RG == kRaggedRows && prm.dev_tab != nullptr) {
        row_tiles = segtab::cap_tiles(prm.dev_rows_cap, prm.tab.n, 128) * (128 / BM);
        prm.dev_map_off = (int32_t)segtab::map128_off(prm.dev_rows_cap, prm.tab.n);
    } else if (RG == kRaggedRows) {
        row_tiles = prm.tab.tile[prm.tab.n];
    }
    const int64_t total = row_tiles * prm.tiles_n * (EPI == kEpiParts ? prm.k_split : 1);
    if (total > (int64_t)INT32_MAX - 8) return fail(FMOE_ELIMIT, "grouped GEMM: %lld tiles exceed the grid limit", (long long)total);
    if (total == 0) return FMOE_OK;
    prm.total_tiles = (int)total;
    std::optional<ProfileScope> prof;
    if (EPI != kEpiParts) prof.emplace(prm.profile_class, prm.profile_work, stream);   // (parts: launch_parts, around both launches)
    grouped_gemm_unaligned_kernel<T, BM, PS, QS, RG, EPI><<<(unsigned)((total + 7) / 8 * 8), kUaThreads, 0, stream>>>(prm);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

// Ragged rows over a device table, prm.k_split parts of prm.split_slabs slabs each: sums into prm.split_ws, and those added up.
template <typename T, int PS> int launch_parts(GemmParams &prm, hipStream_t stream) {
    ProfileScope prof(prm.profile_class, prm.profile_work, stream);
    if (int rc = launch_unaligned_tiles<T, 64, PS, kKC, kRaggedRows, kEpiParts>(prm, kEpiStore, stream)) return rc;
    prm.dev_map_off = (int)segtab::map128_off(prm.dev_rows_cap, prm.tab.n);
    const int64_t places = segtab::cap_tiles(prm.dev_rows_cap, prm.tab.n, 128);
    add_parts_kernel<T><<<dim3((unsigned)(places * 8), (unsigned)ceil_div(prm.n_cols, 256)), kUaThreads, 0, stream>>>(prm);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

template <typename T> int launch_unaligned_typed(GemmParams &prm, int product, int epilogue, hipStream_t stream) {
    const bool low = prm.block_m == 64;
    switch (product) {
        case 5: return launch_parts<T, kKC>(prm, stream);
        case 6: return launch_parts<T, kMC>(prm, stream);
        case 3:
            return low ? launch_unaligned_tiles<T, 64, kKC, kKC, kRaggedRows, kEpiGated>(prm, epilogue, stream)
                       : launch_unaligned_tiles<T, 128, kKC, kKC, kRaggedRows, kEpiGated>(prm, epilogue, stream);
        case 4:
            return low ? launch_unaligned_tiles<T, 64, kMC, kKC, kRaggedRows, kEpiDGated>(prm, epilogue, stream)
                       : launch_unaligned_tiles<T, 128, kMC, kKC, kRaggedRows, kEpiDGated>(prm, epilogue, stream);
        case 0:
            return low ? launch_unaligned_tiles<T, 64, kKC, kKC, kRaggedRows>(prm, epilogue, stream)
                       : launch_unaligned_tiles<T, 128, kKC, kKC, kRaggedRows>(prm, epilogue, stream);
        case 1:
            return low ? launch_unaligned_tiles<T, 64, kMC, kKC, kRaggedRows>(prm, epilogue, stream)
                       : launch_unaligned_tiles<T, 128, kMC, kKC, kRaggedRows>(prm, epilogue, stream);
    }
    return launch_unaligned_tiles<T, 128, kMC, kMC, kRaggedK>(prm, epilogue, stream);
}

}  // namespace

// product: 0 forward, 1 data gradient, 2 weight gradient (with the bias gradient), 3 gated forward, 4 data gradient up to a gated forward's product, 5 and 6 forward
// and data gradient in parts of the contraction.  Ragged rows: prm.block_m (64 or 128)
// is the tile height, for which prm.tab was filled in (a device table serves both).
int launch_mfma_unaligned(gemm::GemmParams &prm, int dtype, int product, int epilogue, hipStream_t stream) {
    if (dtype == FMOE_BF16) return launch_unaligned_typed<__bf16>(prm, product, epilogue, stream);
    if (dtype == FMOE_F16) return launch_unaligned_typed<_Float16>(prm, product, epilogue, stream);
    return fail(FMOE_EINVAL, "grouped GEMM: dtype %d is not a 16-bit float type", dtype);
}

}  // namespace fmoe
