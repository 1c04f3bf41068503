// Grouped forward product Y[seg_e] = act(X[seg_e] . W_e^T + b_e) for few rows per expert, 16- and 32-bit types over a device
// segment table (gfx950): decoding steps, where every weight is read once and meets a handful of rows.
//
// Bound by the weights' way from memory, so nothing is staged: weights and rows go from memory (the rows: L2, where they stay) straight
// into the registers of 16 x 16 x 32 MFMAs (float32: 16 x 16 x 4).  A workgroup of four waves has up to 64 columns of up to 32 rows of one expert; the
// waves take the contraction in turns of one unit, with the next unit's loads under way before the products of the current one, and add
// up their accumulators through LDS in a fixed order.  What it takes to come near the 6.9 TB/s that such loads alone reach here
// (8 experts of 4096 x 14336, 8 rows each: 189 us before, 137 now; of 14336 x 4096: 187 and 142):
//   * a load takes whole lines, 128 bytes of eight rows, and leaves no trace in the caches (6.2 TB/s through them; 64 bytes of
//     sixteen rows, the operands' own shape, read nontemporally: 5.5, as the halves of a line are fetched apart), unless the weights are read
//     again soon and fit there (weights_cached);
//   * the rows' loads, which take as many places in a unit's queue of loads as the weights' do, serve two or four blocks of 16 columns
//     (one block: 362 us for that layer's pass, without the rows' loads 300);
//   * each workgroup of an expert begins its contraction one unit further on than the one before, so that they don't all ask the same
//     channels for the same columns at once (162 -> 142 us for 14336 x 4096); where it begins is its expert's and its columns' own, so that a row's
//     sum, in the order of the units from there on, does not depend on how many rows other experts have;
//   * the compiler may not move a unit's loads behind the products of the one before, which left none in flight at their end.
// Where it is used, and what it measured: use_skinny() in grouped_gemm.hip.
//
// Gated products (HALVES): half of a workgroup's blocks of columns are the gate's and the others the same columns of the linear half, so that the wave that adds up a
// block of the one adds up the other's too.  8-bit integers: see Int8Pair; the sums are integers and exact.  ROUND: the rows come as they are and each workgroup rounds
// its expert's to integers in LDS while its first weights are on their way: see kSkinnyRoundElems.
// The build compiles this file with -DFMOE_SKINNY=<0 plain products|1 gated ones|2 8-bit integers>.
#include "gemm_skinny.hpp"
#include "row_rounding.hpp"
#include "segment_table.hpp"

namespace fmoe {
namespace gemm {
namespace {

constexpr int kSkWaves = 4, kSkThreads = 64 * kSkWaves;
constexpr int kSkRows = 32;   // rows of a pass

// one 16 x 16 block over 64 bytes of contraction; acc as for the 16 x 16 x 32 form
template <typename T> __device__ __forceinline__ void mma_step(f32x4 &acc, const u32x4 &w, const u32x4 &x) { Elem<T>::mma(acc, w, x); }
template <> __device__ __forceinline__ void mma_step<float>(f32x4 &acc, const u32x4 &w, const u32x4 &x) {
    // product j takes element j of every lane's four: contraction elements j, 4 + j, 8 + j and 12 + j of the step
#pragma unroll
    for (int j = 0; j < 4; ++j)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[j]), __uint_as_float(x[j]), acc, 0, 0, 0);
}

template <typename T, bool HALVES> using Params = std::conditional_t<HALVES || IsInt8<T>::value, SkinnyMoreParams, SkinnyParams>;

// COL_BLOCKS: blocks of 16 columns of a workgroup.  APART: an expert's groups of rows have workgroups of their own (see launch).  HALVES: gated.  ROUND: at most
// kSkinnyRoundRows rows in all, of the results' type
template <typename T, int COL_BLOCKS, bool APART, bool HALVES, bool ROUND>
__global__ __launch_bounds__(kSkThreads, COL_BLOCKS == 4 ? 3 : 4) void grouped_gemm_skinny_kernel(const Params<T, HALVES> prm) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only needs the launch stub
    constexpr int EB = (int)sizeof(T), CE = 16 / EB, kLine = 128 / EB;    // elements per lane's load and per line
    typedef std::conditional_t<sizeof(T) == 2, u32x2, u32x4> Vec4;        // four elements
    constexpr bool kInt8 = IsInt8<T>::value;
    typedef typename Elem<T>::Out Out;                                // of the results
    typedef std::conditional_t<sizeof(Out) == 2, u32x2, u32x4> OutVec4;
    constexpr int kCols = COL_BLOCKS * 16 / (HALVES ? 2 : 1);             // columns of a workgroup
    static_assert(!HALVES || (COL_BLOCKS >= 2 && sizeof(T) == 2), "halves: two blocks of columns or more");
    constexpr uint32_t kOutOfRange = 0x80000000u;
    constexpr int kRsrcFlags = 0x00020000;   // raw buffer, 32-bit data format
    typedef const int32_t __attribute__((address_space(4))) *DevTab;    // read-only, uniform: scalar loads
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef const i32x4 __attribute__((address_space(4))) *DevTab4;
    __shared__ f32x4 part[kSkWaves - 1][COL_BLOCKS * 2][64];
    // (16 bytes more than a row: eight rows' pieces at one place of theirs lie in different banks)
    __shared__ __attribute__((aligned(16))) unsigned char rounded[ROUND ? kSkinnyRoundElems + kSkinnyRoundRows * 16 : 16];
    __shared__ uint32_t most_of[kSkinnyRoundRows];

    const DevTab dtab = (DevTab)(uintptr_t)prm.dev_tab;
    int place = __builtin_amdgcn_readfirstlane(blockIdx.x / prm.tiles_n);
    const int tile_n = blockIdx.x - place * prm.tiles_n, n0 = tile_n * kCols, K = prm.k_extent;
    const DevTab4 order = (DevTab4)(dtab + prm.order_off);   // {expert, first row, rows}: of an expert, or (not APART) of a tile of at most 128 rows
    const int live = dtab[APART ? segtab::kLive : segtab::kTiles128];
    if constexpr ((HALVES && !kInt8) || ROUND) {
        const int64_t there = dtab[segtab::kRows];
        if (prm.tail != nullptr && there < prm.tail_rows)
            for (int64_t i = (int64_t)blockIdx.x * kSkThreads + threadIdx.x; i < (prm.tail_rows - there) * prm.tail_elems; i += (int64_t)gridDim.x * kSkThreads)
                ((Out *)prm.tail)[there * prm.tail_elems + i] = (Out)0.f;
    }
    int r0 = 0;   // first row
    i32x4 entry;
    if (APART && place < prm.extra_groups) {
        // A further group of an expert with more rows than one pass takes; the experts come in descending order of their rows
        int i = 0, skip = place;
        for (;; ++i) {
            entry = order[i];   // (there is an expert 0; the ones before have more than kSkRows rows, so `i` is not past the last live one)
            const int groups = (entry[2] - 1) / kSkRows;   // (without rows: 0)
            if (groups == 0) return;
            if (skip < groups) break;
            skip -= groups;
            if (i + 1 >= live) return;
        }
        r0 = (skip + 1) * kSkRows;
    } else {
        place -= prm.extra_groups;
        entry = order[place];   // (asked for together with their number; the launch has as many places as experts can have rows, or as there can be tiles)
        asm volatile("" : "+s"(entry));
        if (place >= live) return;
    }
    const int expert = entry[0], first = entry[1], rows = ROUND ? min(entry[2], kSkinnyRoundRows) : entry[2];
    if (rows == 0) return;
    // where its contraction begins, by expert and columns alone: a row's sum does not depend on the rows that other experts have
    const uint32_t start = __builtin_amdgcn_readfirstlane((uint32_t)expert * (uint32_t)prm.tiles_n + (uint32_t)tile_n);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int lb = lane & 15, hq = lane >> 4;
    // A load takes 128 bytes of eight rows, this lane 16 bytes of row lane % 8 (see pair_to_steps)
    const int chunk = hq | ((lane & 8) >> 1), row8 = lane & 7;

    // weights: rows past the last column lie past the end of the resource and read as zero
    // (gated: past the last of the gate's columns lie the linear half's)
    int ldw = K, ldx = K;    // elements from row to row
    int64_t w_first = ((int64_t)expert * ((HALVES ? 2 : 1) * prm.n_cols) + n0) * K;
    if constexpr (kInt8) {
        ldw = (int)prm.ldw;
        ldx = (int)prm.ldx;
        w_first = expert * prm.w_expert_stride + (int64_t)n0 * ldw;
    }
    const T *W = (const T *)prm.w + w_first;
    const int w_bytes = (min(kCols, prm.n_cols - n0) + (HALVES ? prm.n_cols : 0)) * ldw * EB;
    const __amdgpu_buffer_rsrc_t w_rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(W), 0, w_bytes, kRsrcFlags);
    const uint32_t w_off = (uint32_t)(row8 * ldw * EB + chunk * 16), eight_rows = (uint32_t)(8 * ldw * EB);
    const uint32_t half_rows = HALVES ? (uint32_t)prm.n_cols * (uint32_t)(ldw * EB) : 0u;
    const bool gather = !ROUND && prm.row_index != nullptr;

    // Rows to be rounded: all of the expert's, eight elements at a time, asked for before the first weights.
    constexpr int kPieces = ROUND ? kSkinnyRoundElems / (kLaneElems * kSkThreads) : 1;
    Eight<Out> raw[kPieces];
    const int row_bytes = K * 2 + 16, row_pieces = K * 2 / kLaneElems;   // (K: pairs)
    auto place_of = [&](int i, int &row, int &col) {
        const int p = t + i * kSkThreads;
        row = (int)((uint32_t)p / (uint32_t)row_pieces);
        col = (p - row * row_pieces) * kLaneElems;
        return row < rows;
    };
    if constexpr (ROUND) {
        if (t < kSkinnyRoundRows) most_of[t] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            int row, col;
            bool there = place_of(i, row, col);
            int64_t src = first + row;
            if (prm.row_index != nullptr && there) {   // (a row from nowhere is one of zeros)
                const int64_t idx = prm.row_index[src];
                src = idx < 0 ? -1 : prm.index_div == 1 ? idx : idx / prm.index_div;
                there = src >= 0 && src < prm.x_total_rows;
            }
            raw[i].load((const Out *)prm.x + (there ? src * prm.ldx + col : 0), there ? prm.x_elems - col : 0);
        }
    }
    auto round_rows = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            int row, col;
            if (place_of(i, row, col)) atomicMax(&most_of[row], magnitude_bits<Out>(larger<Out>(0u, raw[i])));   // (a maximum: in any order)
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            int row, col;
            if (place_of(i, row, col)) *(uint2 *)(rounded + row * row_bytes + col) = RowScale(most_of[row]).round(raw[i]);
        }
        __syncthreads();
    };

    // NB blocks of 16 columns from column c0 of the workgroup on times RB blocks of 16 rows from the expert's row r0 on; a unit is LINES times
    // 128 bytes of contraction.  POLICY: of the weights' loads
    auto pass = [&](auto nb_tag, auto rb_tag, auto lines_tag, auto policy_tag, int c0, int r0) {
        constexpr int NB = decltype(nb_tag)::value, RB = decltype(rb_tag)::value, LINES = decltype(lines_tag)::value;
        constexpr int POLICY = decltype(policy_tag)::value;
        static_assert(NB * RB <= 2 * COL_BLOCKS && NB <= kSkWaves, "the waves' sums");
        constexpr int NH = HALVES ? NB / 2 : NB;   // blocks of a half
        struct Unit { u32x4 w[LINES][NB][2], x[LINES][RB][2]; };
        // The rows, in a resource that begins at the pass's first or at the tile's: all of an expert can be more than the 2 GiB that offsets reach (bit
        // 31 marks one as out of range), these are at most 32 or 128 of 4 MiB.  A gathered matrix is less than 2 GiB as a whole.
        const int base = APART ? r0 : 0, base_rows = APART ? min(rows - r0, 16 * RB) : rows;
        const int64_t base_at = (int64_t)first + base;
        const __amdgpu_buffer_rsrc_t x_rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<T *>((const T *)prm.x + (gather ? (int64_t)0 : base_at * ldx)), 0, (int)(gather ? prm.x_total_rows : (int64_t)base_rows) * ldx * EB, kRsrcFlags);
        const __amdgpu_buffer_rsrc_t index_rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<int64_t *>(gather ? prm.row_index + base_at : nullptr), 0, gather ? base_rows * 8 : 0, kRsrcFlags);
        const uint32_t w_base = w_off + (uint32_t)c0 * (uint32_t)(ldw * EB);
        const int n_units = (K + kLine * LINES - 1) / (kLine * LINES);
        const int turn = __builtin_amdgcn_readfirstlane((int)(start % (uint32_t)n_units));   // the unit it begins with
        // (offsets past the contraction, as of every unit past it, have the sign bit set)
        auto line_offset = [&](int unit, int l) -> uint32_t {
            const int at = unit + turn < n_units ? unit + turn : unit + turn - n_units;
            const int k = unit < n_units ? (at * LINES + l) * kLine : K;
            return (uint32_t)(k * EB) | ((uint32_t)(K - 1 - k - chunk * CE) & kOutOfRange);
        };
        auto load_w = [&](Unit &u, int unit) {
#pragma unroll
            for (int l = 0; l < LINES; ++l) {
                const uint32_t at = w_base + line_offset(unit, l);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint32_t block = at + 2 * (n % NH) * eight_rows + (n < NH ? 0u : half_rows);
                    u.w[l][n][0] = __builtin_amdgcn_raw_buffer_load_b128(w_rs, (int)block, 0, POLICY);
                    u.w[l][n][1] = __builtin_amdgcn_raw_buffer_load_b128(w_rs, (int)(block + eight_rows), 0, POLICY);
                }
            }
        };
        Unit a, b;
        int unit = wave;
        // (asked for ahead of the first weights and waited for behind them)
        u32x2 index[RB][2];
#pragma unroll
        for (int y = 0; y < RB; ++y)
#pragma unroll
            for (int h = 0; h < 2; ++h) index[y][h] = __builtin_amdgcn_raw_buffer_load_b64(index_rs, (r0 - base + 16 * y + 8 * h + row8) * 8, 0, 0);
        load_w(a, unit);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (ROUND) round_rows();
        uint32_t x_off[RB][2];
#pragma unroll
        for (int y = 0; y < RB; ++y)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = r0 - base + 16 * y + 8 * h + row8;
                uint32_t src = row;
                bool valid = row < base_rows;
                if (gather) {
                    const uint32_t idx = index[y][h][0];
                    src = prm.div_shift < 0 ? idx : __umulhi(idx, prm.div_mul) >> prm.div_shift;
                    valid = valid && index[y][h][1] == 0 && idx <= (uint32_t)INT32_MAX && (int64_t)src < prm.x_total_rows;
                }
                x_off[y][h] = valid ? src * (uint32_t)(ldx * EB) + chunk * 16 : kOutOfRange;
            }
        f32x4 acc[NB][RB];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int y = 0; y < RB; ++y) acc[n][y] = f32x4{0.f, 0.f, 0.f, 0.f};
        auto load_x = [&](Unit &u, int unit) {
#pragma unroll
            for (int l = 0; l < LINES; ++l) {
                const uint32_t at = line_offset(unit, l);
#pragma unroll
                for (int y = 0; y < RB; ++y) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)   // (both offsets may have the sign bit)
                        if constexpr (ROUND)
                            u.x[l][y][h] = row8 + 8 * h < rows && !(at & kOutOfRange) ? *(const u32x4 *)(rounded + (row8 + 8 * h) * row_bytes + (int)at + chunk * 16)
                                                                                  : u32x4{0u, 0u, 0u, 0u};
                        else u.x[l][y][h] = __builtin_amdgcn_raw_buffer_load_b128(x_rs, (int)((x_off[y][h] + (at & ~kOutOfRange)) | (at & kOutOfRange)), 0, 0);
                }
            }
        };
        auto multiply = [&](Unit &u) {
#pragma unroll
            for (int l = 0; l < LINES; ++l) {
#pragma unroll
                for (int y = 0; y < RB; ++y) pair_to_steps(u.x[l][y][0], u.x[l][y][1]);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    pair_to_steps(u.w[l][n][0], u.w[l][n][1]);
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int y = 0; y < RB; ++y) mma_step<T>(acc[n][y], u.w[l][n][s], u.x[l][y][s]);
                }
            }
        };
        load_x(a, unit);
        while (unit < n_units) {
            load_w(b, unit + kSkWaves);
            load_x(b, unit + kSkWaves);
            __builtin_amdgcn_sched_barrier(0);   // (or the compiler moves the loads behind the products, and none are in flight at their end)
            multiply(a);
            __builtin_amdgcn_sched_barrier(0);
            unit += kSkWaves;
            if (unit >= n_units) break;
            load_w(a, unit + kSkWaves);
            load_x(a, unit + kSkWaves);
            __builtin_amdgcn_sched_barrier(0);
            multiply(b);
            __builtin_amdgcn_sched_barrier(0);
            unit += kSkWaves;
        }
        // the waves' sums in ascending order of the wave; wave n adds column block n's (of both halves)
        __syncthreads();   // (the pass before has read its sums)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            if (wave == n % NH) continue;
#pragma unroll
            for (int y = 0; y < RB; ++y) part[wave - (wave > n % NH ? 1 : 0)][n * RB + y][lane] = acc[n][y];
        }
        __syncthreads();
        auto summed = [&](int n, int y) -> f32x4 {
            f32x4 v = n % NH == 0 ? acc[n][y] : part[0][n * RB + y][lane];
#pragma unroll
            for (int w = 1; w < kSkWaves; ++w)
                v = add_parts<T>(v, w == n % NH ? acc[n][y] : part[w - (w > n % NH ? 1 : 0)][n * RB + y][lane]);
            return v;
        };
#pragma unroll
        for (int n = 0; n < NH; ++n) {
            if (wave != n) continue;
            if constexpr (HALVES || kInt8) {
                // the sums (in integers: under their scales) with the bias, of one half or both
                constexpr int H = HALVES ? 2 : 1;
                const int col = n0 + c0 + 16 * n + 4 * hq;
                if (col >= prm.n_cols) continue;
                const int64_t channel = (int64_t)expert * (H * prm.n_cols) + col;
                float add[H][4] = {}, scale[H][4] = {};
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    if (prm.bias != nullptr) {
                        alignas(16) Out b4[4];
                        *(OutVec4 *)b4 = *(const OutVec4 *)((const Out *)prm.bias + channel + h * prm.n_cols);
#pragma unroll
                        for (int i = 0; i < 4; ++i) add[h][i] = (float)b4[i];
                    }
                    if constexpr (kInt8) __builtin_memcpy(scale[h], prm.w_scale + channel + h * prm.n_cols, 16);
                }
#pragma unroll
                for (int y = 0; y < RB; ++y) {
                    const int row = r0 + 16 * y + lb;
                    const f32x4 sum[2] = {summed(n, y), HALVES ? summed(n + NH, y) : f32x4{}};
                    if (row >= rows) continue;
                    const float s = ROUND ? RowScale(most_of[row]).shown() : kInt8 ? prm.x_scale[first + row] : 1.f;
                    alignas(16) Out res[4];
                    f32x4 pre[H];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[H];
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            if constexpr (kInt8) v[h] = fmaf((float)(int)__float_as_uint(sum[h][i]), s * scale[h][i], add[h][i]);
                            else v[h] = sum[h][i] + add[h][i];
                            pre[h][i] = v[h];
                        }
                        float r = gate_act<sizeof(Out) == 2>(v[0], prm.activation);
                        if constexpr (HALVES) r *= v[1];
                        res[i] = (Out)r;
                    }
                    const int64_t at = (int64_t)(first + row) * prm.n_cols + col;
                    if (HALVES && prm.aux != nullptr) {
#pragma unroll
                        for (int h = 0; h < H; ++h)
                            *(f32x4 *)((float *)prm.aux + 2 * at - col + h * prm.n_cols) = pre[h];
                    }
                    *(OutVec4 *)((Out *)prm.y + at) = *(const OutVec4 *)res;
                }
            } else {
            // acc[n][y][i] is C(row 16 y + lb, column 16 n + 4 hq + i)
            const int col = n0 + c0 + 16 * n + 4 * hq;
            alignas(16) T b4[4] = {};
            if (prm.bias != nullptr && col < prm.n_cols)
                *(Vec4 *)b4 = *(const Vec4 *)((const T *)prm.bias + (int64_t)expert * prm.n_cols + col);
#pragma unroll
            for (int y = 0; y < RB; ++y) {
                const f32x4 v = summed(n, y);
                const int row = r0 + 16 * y + lb;
                if (row >= rows || col >= prm.n_cols) continue;
                alignas(16) T pre[4], res[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = v[i] + (float)b4[i];
                    pre[i] = (T)p;
                    res[i] = (T)apply_act<sizeof(T) == 2>(p, prm.activation);
                }
                const int64_t at = (int64_t)(first + row) * prm.n_cols + col;
                if (prm.aux != nullptr) *(Vec4 *)((T *)prm.aux + at) = *(const Vec4 *)pre;
                *(Vec4 *)((T *)prm.y + at) = *(const Vec4 *)res;
            }
            }
        }
    };
    typedef std::integral_constant<int, 0> Cached;
    typedef std::integral_constant<int, 2> Nontemporal;
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, COL_BLOCKS> All;
    typedef std::integral_constant<int, (COL_BLOCKS < 2 ? COL_BLOCKS : 2)> UpToTwo;
    // (Two units have to fit 168 registers: scratch memory costs launches that never touch it a tenth of their time.  The weights of an
    // expert with several groups are read again, from the caches.)
    if (ROUND || rows <= 16) {
        const std::integral_constant<int, COL_BLOCKS == 1 ? 2 : 1> lines;
        if (prm.weights_cached) pass(All{}, One{}, lines, Cached{}, 0, 0);
        else pass(All{}, One{}, lines, Nontemporal{}, 0, 0);
        return;
    }
    if constexpr (!ROUND) {
    auto up_to_two = [&](int c0) {
        if (rows <= kSkRows && !prm.weights_cached) {
            pass(UpToTwo{}, Two{}, One{}, Nontemporal{}, c0, 0);
        } else if constexpr (APART) {
            pass(UpToTwo{}, Two{}, One{}, Cached{}, c0, r0);
        } else {
            for (int row = 0; row < rows; row += kSkRows) pass(UpToTwo{}, Two{}, One{}, Cached{}, c0, row);
        }
    };
    up_to_two(0);
    constexpr int kNext = HALVES ? 16 : 32;
    if (COL_BLOCKS > 2 && prm.n_cols - n0 > kNext) up_to_two(kNext);
    }
#endif
}

// Column blocks of a workgroup.  More of them share a row's loads; fewer spread a launch, and the long contractions of an expert with
// more than 16 rows, over more workgroups.  us with 1 / 2 / 4 blocks, 16-bit types, equal counts unless said otherwise: 2 experts of 4096
// x 1024, one row each: 9.5 / 13.0 / 19.2; 8 of 1024 x 4096, 8 rows in all: 16.9 / 14.8 / 14.2; 256 of 2048 x 1024, 512: 187 / 163 / 168;
// 8 of 4096 x 14336, 64: 178 / 152 / 137, shares 1 / rank^1.2: 179 / 157 / 146; 64 of 8192 x 2048, 512, such shares: 445 / 400 / 515.  So
// one where two would make fewer workgroups than there are compute units, and four where one expert makes half as many.
// (float32 with 4 loses on skewed counts everywhere: 8 of 2048 x 8192, 192 rows: 183 / 144 / 161.)
template <typename T> int skinny_blocks(const SkinnyParams &prm, int64_t experts, int n_cols, bool gated) {
    const int64_t cus = device_compute_units();
    if (!gated && experts * ceil_div(n_cols, 32) < cus) return 1;
    // (a workgroup's weights in one buffer resource)
    return sizeof(T) == 2 && ceil_div(n_cols, 64) * 2 >= cus && (int64_t)prm.k_extent * 2 * 64 < ((int64_t)1 << 31) ? 4 : 2;
}

template <typename T, bool HALVES = false, bool ROUND = false> int launch(const Params<T, HALVES> &params, int64_t rows_cap, int64_t n_expert, hipStream_t stream) {
    Params<T, HALVES> prm = params;
    // An expert's groups of rows go to workgroups of their own, where the experts come in order of their rows: the further groups first,
    // which leave at once where there are none.  128 experts of 1280 x 1280, 448 rows, 144 of them one expert's: 37 us in turn, 29 apart; 64 of 1280 x
    // 1280 in float32, 900 and 274: 116 and 82.
    // More experts are in no order, and those with rows are found through the map of row tiles, at most as many as there are rows: 8192 experts of 64 x
    // 1024, 8 slots: 9 us on 256 workgroups, where a place for each expert makes 262144 and 71; 2048 of 512 x 512, 64 slots: 9 and 17.
    const bool apart = n_expert <= segtab::kSmallExperts;
    prm.order_off = (int32_t)(apart ? segtab::order_off(rows_cap, n_expert) : segtab::map128_off(rows_cap, n_expert));
    prm.extra_groups = apart ? (int32_t)(rows_cap / kSkRows) : 0;
    const int64_t experts = apart ? std::min(rows_cap, n_expert) : segtab::cap_tiles(rows_cap, n_expert, 128);
    const int blocks = apart ? skinny_blocks<T>(prm, experts, (HALVES ? 2 : 1) * prm.n_cols, HALVES) : 2;
    prm.tiles_n = (int)ceil_div(prm.n_cols, 16 * blocks / (HALVES ? 2 : 1));
    const int64_t grid = (experts + prm.extra_groups) * prm.tiles_n;
    if (grid > (int64_t)INT32_MAX) return fail(FMOE_ELIMIT, "grouped GEMM: grid of %lld workgroups", (long long)grid);
    if (!apart) grouped_gemm_skinny_kernel<T, 2, false, HALVES, ROUND><<<(unsigned)grid, kSkThreads, 0, stream>>>(prm);
    else if (blocks == 2) grouped_gemm_skinny_kernel<T, 2, true, HALVES, ROUND><<<(unsigned)grid, kSkThreads, 0, stream>>>(prm);
    else if (blocks == 1) { if constexpr (!HALVES) grouped_gemm_skinny_kernel<T, 1, true, false, ROUND><<<(unsigned)grid, kSkThreads, 0, stream>>>(prm); }
    else if constexpr (sizeof(T) == 2) grouped_gemm_skinny_kernel<T, 4, true, HALVES, ROUND><<<(unsigned)grid, kSkThreads, 0, stream>>>(prm);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

}  // namespace

#if FMOE_SKINNY == 0
int launch_skinny(const SkinnyParams &prm, int dtype, int64_t rows_cap, int64_t n_expert, hipStream_t stream) {
    FMOE_REQUIRE(dtype == FMOE_BF16 || dtype == FMOE_F16 || dtype == FMOE_F32, "grouped GEMM: dtype %d is not a 16- or 32-bit float type", dtype);
    if (dtype == FMOE_F32) return launch<float>(prm, rows_cap, n_expert, stream);
    return dtype == FMOE_BF16 ? launch<__bf16>(prm, rows_cap, n_expert, stream) : launch<_Float16>(prm, rows_cap, n_expert, stream);
}
#elif FMOE_SKINNY == 1
int launch_skinny_gated(const SkinnyMoreParams &prm, int dtype, int64_t rows_cap, int64_t n_expert, hipStream_t stream) {
    FMOE_REQUIRE(dtype == FMOE_BF16 || dtype == FMOE_F16, "grouped GEMM: dtype %d is not a 16-bit float type", dtype);
    return dtype == FMOE_BF16 ? launch<__bf16, true>(prm, rows_cap, n_expert, stream) : launch<_Float16, true>(prm, rows_cap, n_expert, stream);
}
#elif FMOE_SKINNY == 2
int launch_skinny_int8(const SkinnyMoreParams &prm, int dtype, bool gated, int64_t rows_cap, int64_t n_expert, hipStream_t stream) {
    auto go = [&](auto pair) {
        using Pair = decltype(pair);
        if (prm.x_scale == nullptr) return gated ? launch<Pair, true, true>(prm, rows_cap, n_expert, stream) : launch<Pair, false, true>(prm, rows_cap, n_expert, stream);
        return gated ? launch<Pair, true>(prm, rows_cap, n_expert, stream) : launch<Pair>(prm, rows_cap, n_expert, stream);
    };
    if (dtype == FMOE_F32) return go(Int8Pair<float>{});
    return dtype == FMOE_BF16 ? go(Int8Pair<__bf16>{}) : go(Int8Pair<_Float16>{});
}
#else
#error "FMOE_SKINNY must be 0, 1 or 2"
#endif

}  // namespace gemm
}  // namespace fmoe
