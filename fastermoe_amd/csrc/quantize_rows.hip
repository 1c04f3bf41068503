// Rows rounded to 8-bit integers, each under a scale of its own (gfx950):
//
//   s = max(fl32(max|x| / 127), 2^-126)        q = x / s to the nearest integer, ties to even, of the exact quotient
//
// A row with an infinity or a NaN has the scale NaN and zeros, so that whatever is made of it is NaN.
//
// The rounding itself: row_rounding.hpp.
//
// A lane takes eight elements at a time.  A row that fits the registers of its wave, or, longer (or where rows are few), of its workgroup's four waves, is read once; a
// longer one is read again, from the caches.  Bound by memory, and next by 7 instructions an element (18 with a conversion and a correction for each: 354 us for 32768
// rows of 14336 in bfloat16, 250 now, 5.6 TB/s); few rows by the chain of a load, the row's largest and a store (1018 rows of 1302: 4.3 us).
#include "common.hpp"
#include "grouped_gemm.hpp"
#include "row_rounding.hpp"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kBlock = 256, kWaves = kBlock / kWave;
constexpr int64_t kManyRows = 1024;   // a row's pieces times this

struct Params {
    const void *x;
    const int64_t *row_index;    // or null: row r is read from row row_index[r] / index_div of x
    int64_t index_div, x_rows, ldx;
    int8_t *q;                   // rows of ldq bytes, zeros from d on
    float *scale;
    const int32_t *table;        // or null
    int64_t rows, ldq;
    int d, dq;                   // features; features rounded up to whole pieces
    uint8_t *tail;               // or null: rows of tail_bytes bytes, those behind the table's become zeros
    int64_t tail_bytes;
};

// ROW_WAVES: waves that share a row, 1 or all of the workgroup; NV: pieces of a lane that stay in registers (0: the row is read twice)
template <typename T, int ROW_WAVES, int NV>
__global__ __launch_bounds__(kBlock) void quantize_rows_kernel(const Params prm) {
    __shared__ uint32_t most_of[kWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t live = prm.table ? min((int64_t)prm.table[segtab::kRows], prm.rows) : prm.rows;
    const int64_t row = ROW_WAVES == 1 ? (int64_t)blockIdx.x * kWaves + wave : (int64_t)blockIdx.x;
    if (row >= live) {   // (ROW_WAVES > 1: the whole workgroup)
        if (prm.tail && row < prm.rows) {
            uint8_t *at = prm.tail + row * prm.tail_bytes;   // (bytes: rows of any length)
            for (int64_t i = ROW_WAVES == 1 ? lane : (int)threadIdx.x; i < prm.tail_bytes; i += ROW_WAVES * kWave) at[i] = 0;
        }
        return;
    }
    int64_t src = row;
    bool there = true;
    if (prm.row_index) {
        const int64_t idx = prm.row_index[row];
        src = idx < 0 ? -1 : prm.index_div == 1 ? idx : idx / prm.index_div;
        there = src >= 0 && src < prm.x_rows;
    }
    const T *x = (const T *)prm.x + (there ? src : 0) * prm.ldx;
    int8_t *q = prm.q + row * prm.ldq;
    const int first = ((ROW_WAVES == 1 ? 0 : wave * kWave) + lane) * kLaneElems;
    constexpr int kStep = ROW_WAVES * kWave * kLaneElems;
    const int d = there ? prm.d : 0;   // (a row from nowhere is one of zeros)
    Eight<T> e[NV ? NV : 1];
    uint32_t most = 0;
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) e[i].load(x + first + i * kStep, d - first - i * kStep);
#pragma unroll
        for (int i = 0; i < NV; ++i) most = larger<T>(most, e[i]);
    } else {
        for (int c = first; c < d; c += kStep) {
            e[0].load(x + c, d - c);
            most = larger<T>(most, e[0]);
        }
    }
    most = magnitude_bits<T>(most);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, kWave));
    if (ROW_WAVES > 1) {
        if (lane == 0) most_of[wave] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = max(most, most_of[w]);
    }
    const RowScale scale(most);
    if (first == 0) prm.scale[row] = scale.shown();
    auto store = [&](int c, const Eight<T> &piece) {
        const uint2 w = scale.round(piece);
        if (c < prm.dq) *(uint2 *)(q + c) = w;
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store(first + i * kStep, e[i]);
    } else {
        for (int c = first; c < prm.dq; c += kStep) {
            e[0].load(x + c, d - c);
            store(c, e[0]);
        }
    }
}

template <typename T> int launch(const Params &prm, hipStream_t stream) {
    auto go = [&](auto waves, auto nv) {
        constexpr int W = decltype(waves)::value;
        const int64_t grid = W == 1 ? ceil_div(prm.rows, kWaves) : prm.rows;
        quantize_rows_kernel<T, W, decltype(nv)::value><<<(unsigned)grid, kBlock, 0, stream>>>(prm);
    };
    typedef std::integral_constant<int, 0> Again;
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    typedef std::integral_constant<int, 8> Eight8;
    const int pieces = (int)ceil_div(prm.dq, kWave * kLaneElems);   // of a wave
    // A wave to a row where there are rows enough for that to fill the card, and its pieces are few.  us with a wave / a workgroup to a row, in a graph, bfloat16: rows of
    // 1024, 1024 of them: 3.9 / 3.6, 2048: 4.1 / 4.6, 32768: 17.8 / 30.1; of 2048, 2048: 6.0 / 5.0, 4096: 7.4 / 7.3, 32768: 32.5 / 36.4; of 4096, 2048: 9.6 / 6.8, 32768: 77 / 70;
    // float32: of 1024, 2048: 3.4 / 4.0; of 2048, 4096: 6.9 / 7.8, 32768: 57 / 55; of 4096, 32768: 119 / 116.
    const bool many = prm.rows >= kManyRows * pieces;
    if (pieces <= 1) go(One{}, One{});
    else if (pieces <= 2 && many) go(One{}, Two{});
    else if (pieces <= 4 && many) go(One{}, Four{});
    else if (pieces <= 4) go(Four{}, One{});
    else if (pieces <= 8) go(Four{}, Two{});
    else if (pieces <= 16) go(Four{}, Four{});
    else if (pieces <= 32) go(Four{}, Eight8{});
    else go(Four{}, Again{});
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_quantize_rows(const void *x, int64_t ldx, const int64_t *row_index, int64_t index_div, int64_t x_rows, void *q, int64_t ldq,
                                  void *scale, const void *segment_table, void *tail, int64_t tail_bytes, int64_t rows, int64_t row_elems, int dtype,
                                  void *stream) {
    const char *who = "fmoe_quantize_rows";
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who, dtype);
    FMOE_REQUIRE(rows >= 0 && row_elems >= 0 && x_rows >= 0, "%s: bad sizes", who);
    FMOE_REQUIRE(row_index == nullptr || index_div >= 1, "%s: index_div=%lld", who, (long long)index_div);
    FMOE_REQUIRE(row_index != nullptr || x_rows >= rows, "%s: %lld rows of %lld", who, (long long)rows, (long long)x_rows);
    FMOE_REQUIRE(tail == nullptr || (segment_table != nullptr && tail_bytes >= 0), "%s: a tail goes with a segment table", who);
    if (rows > kMostThreads / kBlock || row_elems > (int64_t)(1 << 28)) return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    const int64_t whole = ceil_div(row_elems, 16) * 16;
    FMOE_REQUIRE(ldq >= whole && ldq % 16 == 0 && aligned16(q), "%s: rows of 8-bit integers begin on 16 bytes, at least %lld apart", who, (long long)whole);
    if (rows == 0) return FMOE_OK;
    FMOE_REQUIRE((x || row_elems == 0 || x_rows == 0) && (q || row_elems == 0) && scale, "%s: NULL pointer", who);
    const Params prm{x, row_index, index_div, x_rows, ldx, (int8_t *)q, (float *)scale, (const int32_t *)segment_table, rows, ldq, (int)row_elems,
                     (int)whole, (uint8_t *)tail, tail_bytes};
    if (dtype == FMOE_F32) return launch<float>(prm, (hipStream_t)stream);
    return dtype == FMOE_BF16 ? launch<__bf16>(prm, (hipStream_t)stream) : launch<_Float16>(prm, (hipStream_t)stream);
}
