// C entry point of the FP8 product with a fused epilogue, and its kernel for few rows (single tokens and a handful of them).
#include "activation.cuh"
#include "gemm_call.h"
#include "linear_call.h"

#include <algorithm>
#include <atomic>

namespace msamp {

typedef int rows_v8i __attribute__((ext_vector_type(8)));
typedef float rows_v4f __attribute__((ext_vector_type(4)));

constexpr int kMostK = 1 << 26;    // offsets inside the 64 rows of a workgroup are 32 bits
constexpr long long kMostRows = 65535LL * 64;    // workgroups in a grid's second dimension, of 64 rows (so many are never taken by less)

// Up to 16 * MB rows of D per workgroup, RB blocks of 16 columns of it.  The weight a is read once and everything else is small: what
// bounds it is the weight's way from memory, and for the smallest weights the latency of a launch, of a load and of the sum.
//
// A wavefront takes whole slices of K (128 codes of a row) by itself, every `waves`-th.  A load covers eight rows, eight lanes side by
// side to the 128 bytes of a row: with the rows side by side instead, as the MFMA's operand has them, 16 bytes a clock came through a
// compute unit's L1, a quarter of this.  The codes are turned in a part of the LDS that is the wavefront's own (16-byte chunk c
// of row r lies at c ^ (r % 8)), and the loads of its next slice are on their way as soon as they are there.  The wavefronts add up
// through LDS, and a thread then has eight neighbouring columns of a row, whose gate, residual and bias it has asked for before the
// first slice.
// bfloat16, 1 x 4096 -> 11008 with a gate: 9.5 us, 45 MB of weight at 4.8 TB/s; 48 x 4096 -> 12288 with a bias and GELU: 12.0 us.
// WHOLE: 16-byte accesses fit the rows of all operands and outputs, and K is whole chunks.
template <typename OT, int MB, int RB, bool WHOLE>
__global__ __launch_bounds__(512, 2) void fused_rows_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ b, OT* D, int rows, int cols,
                                                            int K, const float* __restrict__ a_scale_inv, const float* __restrict__ b_scale_inv,
                                                            Epilogue ep) {
    // a wavefront's codes, [RB + MB][16 rows][128]; behind them, over the same memory, the parts of the sum, [wavefronts][RB][MB][64]
    extern __shared__ __attribute__((aligned(16))) float4 part[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    uint8_t* const own = reinterpret_cast<uint8_t*>(part) + wave * ((RB + MB) * 2048);
    const int col0 = blockIdx.x * (16 * RB), row0 = blockIdx.y * (16 * MB);
    const int slices = (K + kBK - 1) / kBK;

    // this thread's eight outputs (the host launches a thread for each at least)
    constexpr int kEights = 2 * RB;    // of a row
    const bool has = threadIdx.x < 16 * MB * kEights;
    const int seg = threadIdx.x % kEights, rr = threadIdx.x / kEights % (16 * MB);
    const int row = row0 + rr, col = col0 + seg * 8;
    const bool row_in = has && row < rows;
    const int valid = row_in ? cols - col : 0;
    EpilogueInputs<OT> in;
    epilogue_fetch<OT, WHOLE>(ep, row, col, valid, in);
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = -0.0f;    // (fma(x, y, -0) is x * y to the bit)
    if (ep.bias != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) bias[e] = epilogue_bias(ep, col + e);
    }
    const float alpha = *a_scale_inv * *b_scale_inv;

    // (rows past the end are clamped: their products land in outputs that are not stored)
    const uint8_t* const a0 = a + static_cast<size_t>(col0) * K;
    const uint8_t* const b0 = b + static_cast<size_t>(row0) * K;
    const int r_lane = lane >> 3, chunk = lane & 7;
    uint32_t at[RB + MB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < RB + MB; ++i)
            at[i][h] = static_cast<uint32_t>(i < RB ? min(i * 16 + h * 8 + r_lane, cols - 1 - col0) : min((i - RB) * 16 + h * 8 + r_lane, rows - 1 - row0)) * K;
    }
    // 16 codes of a row from k on, zeros past its end
    auto codes = [&](const uint8_t* p, uint32_t off, int k) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
            // (a load there reads the row's last 16, and what it read is dropped when it is used)
            return *reinterpret_cast<const uint4*>(p + (off + static_cast<uint32_t>(min(k, K - 16))));
        } else {
            // rows that begin anywhere
            if (k + 16 <= K) return reinterpret_cast<const Anywhere16<uint8_t>*>(p + (off + static_cast<uint32_t>(k)))->v;
            union {
                uint8_t e[16];
                uint4 w;
            } u;
            u.w = make_uint4(0, 0, 0, 0);
            for (int i = 0; i < 16; ++i)
                if (k + i < K) u.e[i] = p[off + static_cast<uint32_t>(k + i)];
            return u.w;
        }
    };
    // Workgroups begin with different slices: all of them at the same one, whose rows of b lie a multiple of K apart, were at the same
    // channel of their L2.
    const int turn = static_cast<int>(blockIdx.x * 5u % static_cast<uint32_t>(slices));
    auto k_of = [&](int i) __attribute__((always_inline)) { return (i + turn < slices ? i + turn : i + turn - slices) * kBK + chunk * 16; };
    uint4 q[RB + MB][2];
    auto fetch = [&](int i) __attribute__((always_inline)) {
        const int k = k_of(i);
#pragma unroll
        for (int n = 0; n < RB + MB; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) q[n][h] = codes(n < RB ? a0 : b0, at[n][h], k);
    };
    rows_v4f acc[RB][MB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[r][m] = rows_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int l16 = lane & 15, g4 = lane >> 4;
    if (wave < slices) fetch(wave);
    for (int i = wave; i < slices; i += waves) {
        const bool inside = !WHOLE || k_of(i) < K;
#pragma unroll
        for (int n = 0; n < RB + MB; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<uint4*>(own + n * 2048 + (h * 8 + r_lane) * 128 + ((chunk ^ r_lane) << 4)) = inside ? q[n][h] : make_uint4(0, 0, 0, 0);
        if (i + waves < slices) fetch(i + waves);
        // (the rows are this wavefront's own and the LDS serves its requests in order: only the compiler has to keep them so)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        rows_v8i f[RB + MB];
#pragma unroll
        for (int n = 0; n < RB + MB; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 c = *reinterpret_cast<const uint4*>(own + n * 2048 + l16 * 128 + (((2 * g4 + h) ^ (l16 & 7)) << 4));
                f[n][4 * h] = c.x, f[n][4 * h + 1] = c.y, f[n][4 * h + 2] = c.z, f[n][4 * h + 3] = c.w;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");    // (and the next slice's codes behind these reads)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int m = 0; m < MB; ++m)
                acc[r][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f[r], f[RB + m], acc[r][m], 0, 0, 0, 0, 0, 0);
    }
    __syncthreads();    // every wavefront is through with its codes
    // lane l of a block of 16 x 16 has the columns 4 * (l / 16) .. + 3 of row l % 16
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m)
            part[((wave * RB + r) * MB + m) * 64 + lane] = make_float4(acc[r][m][0], acc[r][m][1], acc[r][m][2], acc[r][m][3]);
    __syncthreads();
    if (!has) return;    // (the threads of a block of columns, four side by side, stay or go together)
    float v[8] = {};
    for (int w = 0; w < waves; ++w) {
        const float4* p = part + ((w * RB + seg / 2) * MB + rr / 16) * 64 + (seg & 1) * 32 + (rr & 15);
        const float4 lo = p[0], hi = p[16];
        v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
        v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
    }
    with_activation(ep.act, [&](auto act) __attribute__((always_inline)) {
        epilogue_eight<decltype(act)::value, OT, WHOLE>(ep, D, cols, alpha, v, bias, row, col, valid, row_in, in);
    });
}

template <typename OT, int MB, int RB, bool WHOLE>
static int launch_rows(const msamp_gemm_fused_args& a, const Epilogue& ep, hipStream_t st) {
    const int rows = static_cast<int>(a.n), cols = static_cast<int>(a.m), K = static_cast<int>(a.k);
    constexpr int kThreads = 16 * MB * 2 * RB;    // outputs by eights
    static_assert(kThreads <= 512, "a thread for each");
    const int waves = std::max((kThreads + 63) / 64, std::min(8, (K + kBK - 1) / kBK));
    constexpr int kOwn = std::max((RB + MB) * 2048, RB * MB * 1024);    // of a wavefront: codes, then its part of the sum
    const size_t smem = static_cast<size_t>(waves) * kOwn;
    const dim3 grid((cols + 16 * RB - 1) / (16 * RB), (rows + 16 * MB - 1) / (16 * MB));
    const auto kern = fused_rows_kernel<OT, MB, RB, WHOLE>;
    static std::atomic<bool> configured{false};    // setting the attribute twice is harmless
    if (!configured.load(std::memory_order_acquire)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 8 * kOwn);
        if (e != hipSuccess) return hip_fail(e, "hipFuncSetAttribute(fused_rows_kernel)");
        configured.store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL(kern, grid, dim3(64 * waves), smem, st, a.a, a.b, static_cast<OT*>(a.d), rows, cols, K, a.a_scale_inv, a.b_scale_inv, ep);
    MSAMP_CHECK_LAUNCH("fused_rows_kernel");
    return MSAMP_OK;
}

// Blocks of 16 columns to a workgroup: as many as leave a workgroup to each compute unit, at most four.  b is read by every workgroup,
// so fewer of them cost less, while all compute units have one.  us with 1, 2, 3 and 4 blocks, bfloat16 with a gate, on 256 compute units:
//   48 x 4096 -> 12288 (3 blocks a unit)  13.7, 13.0, 11.6, 12.1    64 x 4096 -> 11008 (2.7)  15.2, 15.4, 12.3, 12.9
//   33 x 4096 -> 16384 (4)                16.3, 14.2, 17.7, 14.1    48 x 11008 -> 4096 (1)    12.0, 13.9, 16.3, 18.8
// the same with the weights of twelve layers in turn, so that they come from memory:
//   1 x 4096 -> 11008 (2.7)               11.1, 11.8, 10.5, 10.7    1 x 11008 -> 4096 (1)     11.9, 12.8, 14.8, 18.1
//   1 x 4096 -> 12288 (3)                 11.9, 12.1, 11.3, 11.4    16 x 4096 -> 11008 (2.7)  11.8, 12.8, 10.7, 11.1
static int column_blocks(long long cols) {
    return static_cast<int>(std::min<long long>(4, ((cols + 15) / 16 + cu_count() - 1) / cu_count()));
}
// More than 64 rows are several workgroups in the other direction, and the weight is read for each of them; the tile kernels need it once
// but take a slice of K after the other with few of them at work.  us here | in tiles, for so many rows:
//   4096 -> 4096    80 11.0 | 17.2   192 15.2 | 17.9   256 19.4 | 17.9       1024 -> 1024    80 3.8 | 8.7   512 5.2 | 8.9
//   11008 -> 4096   80 22.5 | 33.6   192 34.1 | 36.1   256 43.9 | 36.8       8192 -> 512     80 9.3 | 26.3  512 12.5 | 27.4
//   2048 -> 8192    80 10.8 | 14.1   128 11.6 | 14.6   192 16.6 | 14.7       4096 -> 11008   80 21.5 | 18.0
static bool takes_few_rows(long long rows, long long cols) {
    if (rows <= MSAMP_FUSED_ROWS) return true;
    const long long rb = column_blocks(cols), workgroups = (cols + 16 * rb - 1) / (16 * rb) * ((rows + 63) / 64);
    return rb <= 2 && workgroups * (rb + 4) <= 16LL * cu_count();
}

// A checkpoint's blocks are 32 columns, which lie in one workgroup.
template <typename OT, int MB>
static int run_rows_of(const msamp_gemm_fused_args& a, const Epilogue& ep, hipStream_t st) {
    const bool keeps = ep.z_codes != nullptr || ep.gate_codes != nullptr;
    const int want = column_blocks(a.m);
    if (!ep.vec || a.k % 16 != 0 || !aligned(a.a, 16) || !aligned(a.b, 16)) return launch_rows<OT, MB, 2, false>(a, ep, st);
    if (want >= (keeps ? 3 : 4)) return launch_rows<OT, MB, 4, true>(a, ep, st);
    if (want == 3) return launch_rows<OT, MB, 3, true>(a, ep, st);
    if (want == 2 || keeps) return launch_rows<OT, MB, 2, true>(a, ep, st);
    return launch_rows<OT, MB, 1, true>(a, ep, st);
}
template <typename OT>
static int run_rows(const msamp_gemm_fused_args& a, const Epilogue& ep, hipStream_t st) {
    if (a.n <= 16) return run_rows_of<OT, 1>(a, ep, st);
    if (a.n <= 32) return run_rows_of<OT, 2>(a, ep, st);
    if (a.n <= 48) return run_rows_of<OT, 3>(a, ep, st);
    return run_rows_of<OT, 4>(a, ep, st);
}

// Of `rows` rows in tiles, how many to take in a launch of their own, in front of the others.  A last round of large tiles that leaves most
// compute units idle costs as much as a full one; small tiles, two to a compute unit, take what is left over in two thirds of that
// while they are a single round.  us in two launches | in one, bfloat16, `left` small tiles left over:
//   12710 x 1200 -> 4304   340 left  104.0 | 108.9    13481 x 1200 -> 4304   544  112.3 | 108.2    4289 x 4096 -> 4096   64  65.6 | 86.6
//    9000 x 4096 -> 4096   224       119.6 | 136.6    14325 x 4096 -> 4096   512  183.3 | 186.5    6952 x 4096 -> 4096  736  95.6 | 94.4
//   33985 x 4096 -> 4096   320       419.6 | 425.0     9000 x 11008 -> 4096  224  279.8 | 321.5    5018 x 4096 -> 11008 516 203.8 | 201.8
static long long rows_in_front(long long rows, int m, int k) {
    const int NR = static_cast<int>(rows);
    if (k <= kBK || takes_paired_tiles(NR, m, k) || takes_small_tiles(NR, m, k)) return rows;
    const long long cols = (m + kDmaTile - 1) / kDmaTile, tiles = (rows + kDmaTile - 1) / kDmaTile * cols;
    const long long whole = tiles / cu_count() * cu_count() / cols * kDmaTile, rest = rows - whole;
    if (whole <= 0 || rest <= 0) return rows;
    constexpr int kSmall = kDmaTile / 2;
    return (rest + kSmall - 1) / kSmall * ((m + kSmall - 1) / kSmall) <= 2LL * cu_count() ? whole : rows;
}

// Rows of k codes, one behind the other in memory, to rows of whole 16-byte chunks with zeros behind the last code; the rows of a and then
// those of b.  A workgroup takes as many rows at a time as its threads have chunks for, or one.  45 and 16 MB of codes: 27 us, 4.5 TB/s
// read and written.
constexpr int kPadThreads = 256;
__global__ __launch_bounds__(kPadThreads) void pad_codes_kernel(const uint8_t* __restrict__ a, long long a_rows, uint8_t* __restrict__ a_out,
                                                                const uint8_t* __restrict__ b, long long rows, uint8_t* __restrict__ b_out, int k) {
    const int chunks = (k + 15) / 16, per = min(chunks, kPadThreads);
    const int mine = threadIdx.x / per;
    const long long row = static_cast<long long>(blockIdx.x) * (kPadThreads / per) + mine;
    if (mine >= kPadThreads / per || row >= rows) return;
    const uint8_t* in = row < a_rows ? a + row * k : b + (row - a_rows) * k;
    uint8_t* out = row < a_rows ? a_out + row * (chunks * 16LL) : b_out + (row - a_rows) * (chunks * 16LL);
    for (int c = threadIdx.x % per; c < chunks; c += per) {
        uint4 v;
        if (c * 16 + 16 <= k) {
            v = reinterpret_cast<const Anywhere16<uint8_t>*>(in + c * 16)->v;
        } else {
            union {
                uint8_t e[16];
                uint4 w;
            } u;
            u.w = make_uint4(0, 0, 0, 0);
            for (int i = 0; c * 16 + i < k; ++i) u.e[i] = in[c * 16 + i];
            v = u.w;
        }
        *reinterpret_cast<uint4*>(out + c * 16) = v;
    }
}

}    // namespace msamp

using namespace msamp;

extern "C" int msamp_fp8_gemm_fused_pitch(long long m, long long n, long long k, long long* pitch) {
    MSAMP_REQUIRE(m > 0 && n > 0 && k > 0, MSAMP_ERR_SHAPE, "msamp_fp8_gemm_fused_pitch: m=%lld n=%lld k=%lld", m, n, k);
    MSAMP_REQUIRE(pitch != nullptr, MSAMP_ERR_NULL, "msamp_fp8_gemm_fused_pitch: null pointer");
    *pitch = takes_few_rows(n, m) ? k : (k + 15) / 16 * 16;
    return MSAMP_OK;
}

extern "C" int msamp_pad_codes(const uint8_t* a, long long a_rows, uint8_t* a_out, const uint8_t* b, long long b_rows, uint8_t* b_out, long long k,
                               msamp_stream_t stream) {
    MSAMP_REQUIRE(a_rows >= 0 && b_rows >= 0 && k > 0 && k <= kMostK, MSAMP_ERR_SHAPE, "msamp_pad_codes: %lld and %lld rows of %lld", a_rows, b_rows, k);
    MSAMP_REQUIRE((a && a_out) || a_rows == 0, MSAMP_ERR_NULL, "msamp_pad_codes: null pointer");
    MSAMP_REQUIRE((b && b_out) || b_rows == 0, MSAMP_ERR_NULL, "msamp_pad_codes: null pointer");
    MSAMP_REQUIRE(aligned(a_out, 16) && aligned(b_out, 16), MSAMP_ERR_ALIGNMENT, "msamp_pad_codes: outputs must be 16-byte aligned");
    const int chunks = static_cast<int>((k + 15) / 16), per = std::min(chunks, kPadThreads);
    const long long rows = a_rows + b_rows, rows_at_once = kPadThreads / per;
    if (rows == 0) return MSAMP_OK;
    const long long blocks = (rows + rows_at_once - 1) / rows_at_once;
    MSAMP_REQUIRE(blocks <= 0x7fffffffLL, MSAMP_ERR_SHAPE, "msamp_pad_codes: %lld rows", rows);
    hipLaunchKernelGGL(pad_codes_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kPadThreads), 0, static_cast<hipStream_t>(stream), a, a_rows, a_out, b, rows, b_out, static_cast<int>(k));
    MSAMP_CHECK_LAUNCH("pad_codes_kernel");
    return MSAMP_OK;
}

int msamp::check_gemm_fused(const msamp_gemm_fused_args& a) {
    const int dt = static_cast<int>(a.d_dtype);
    MSAMP_REQUIRE(is_hp(dt), MSAMP_ERR_DTYPE, "msamp_fp8_gemm_fused: d_dtype %d", dt);
    MSAMP_REQUIRE(a.bias == nullptr || is_hp(static_cast<int>(a.bias_dtype)), MSAMP_ERR_DTYPE, "msamp_fp8_gemm_fused: bias_dtype %d",
                  static_cast<int>(a.bias_dtype));
    MSAMP_REQUIRE(a.activation >= MSAMP_ACT_NONE && a.activation <= MSAMP_ACT_SILU, MSAMP_ERR_DTYPE, "msamp_fp8_gemm_fused: activation %d",
                  static_cast<int>(a.activation));
    MSAMP_REQUIRE(a.m > 0 && a.n > 0 && a.k > 0 && a.m <= 0x7fffff00LL && a.n <= 0x7fffff00LL && a.k <= kMostK, MSAMP_ERR_SHAPE,
                  "msamp_fp8_gemm_fused: m=%lld n=%lld k=%lld", static_cast<long long>(a.m), static_cast<long long>(a.n), static_cast<long long>(a.k));
    MSAMP_REQUIRE(a.a && a.a_scale_inv && a.b && a.b_scale_inv && a.d, MSAMP_ERR_NULL, "msamp_fp8_gemm_fused: null pointer");
    MSAMP_REQUIRE((a.z_codes == nullptr) == (a.z_exponents == nullptr) && (a.gate_codes == nullptr) == (a.gate_exponents == nullptr) &&
                      (a.gate_codes == nullptr || a.gate != nullptr),
                  MSAMP_ERR_NULL, "msamp_fp8_gemm_fused: a checkpoint is codes and exponents, of a gate that is there");
    MSAMP_REQUIRE(aligned(a.z_codes, 16) && aligned(a.gate_codes, 16), MSAMP_ERR_ALIGNMENT, "msamp_fp8_gemm_fused: codes must be 16-byte aligned");
    MSAMP_REQUIRE((a.gate == nullptr || a.n == 1 || a.gate_stride >= a.m) && (a.residual == nullptr || a.n == 1 || a.residual_stride >= a.m),
                  MSAMP_ERR_SHAPE, "msamp_fp8_gemm_fused: rows of the gate or the residual overlap");
    return MSAMP_OK;
}

extern "C" int msamp_fp8_gemm_fused(const msamp_gemm_fused_args* args, msamp_stream_t stream) {
    MSAMP_REQUIRE(args != nullptr, MSAMP_ERR_NULL, "msamp_fp8_gemm_fused: null pointer");
    const msamp_gemm_fused_args& a = *args;
    const int rc = check_gemm_fused(a), dt = static_cast<int>(a.d_dtype);
    if (rc != MSAMP_OK) return rc;
    const size_t size = hp_size(dt);
    Epilogue ep = {};
    ep.bias = a.bias, ep.bias_dt = static_cast<int>(a.bias_dtype), ep.act = static_cast<int>(a.activation);
    ep.gate = a.gate, ep.gate_ld = a.gate_stride, ep.residual = a.residual, ep.residual_ld = a.residual_stride;
    ep.z_codes = a.z_codes, ep.z_exponents = a.z_exponents, ep.gate_codes = a.gate_codes, ep.gate_exponents = a.gate_exponents;
    // (the tile kernels' offsets from a wave's first row are 31 bits: 128 rows)
    constexpr long long kLongest = 1LL << 21;
    ep.vec = a.m % 8 == 0 && a.m < kLongest && a.gate_stride < kLongest && a.residual_stride < kLongest && aligned(a.d, 16) && aligned(a.gate, 16) && aligned(a.residual, 16) &&
             (a.gate == nullptr || a.gate_stride * size % 16 == 0) && (a.residual == nullptr || a.residual_stride * size % 16 == 0);
    ep.stream = static_cast<size_t>(a.n) * a.m * size >= (size_t(192) << 20);
    hipStream_t st = static_cast<hipStream_t>(stream);
    // The tile kernels fetch 16 bytes of a row at a time, at 32-bit offsets: a weight of 4 GiB and more is left to the other kernel, as
    // are rows that begin anywhere.  A longer x is taken in stretches of rows, and so is one of more rows than the other kernel's
    // grid has in its second dimension.
    const bool tiles = !takes_few_rows(a.n, a.m) && a.m * a.k < (1LL << 32) && a.k % 16 == 0 && aligned(a.a, 16) && aligned(a.b, 16);
    const long long most = tiles ? ((1LL << 32) - 1) / a.k / 16 * 16 : kMostRows;
    const size_t pitch = ckpt_pitch(static_cast<int>(a.m));
    for (long long r = 0, rows; r < a.n; r += rows) {
        rows = std::min(most, a.n - r);
        if (tiles) rows = rows_in_front(rows, static_cast<int>(a.m), static_cast<int>(a.k));
        Epilogue e = ep;
        auto byte = [](const void* p, long long n) { return p == nullptr ? nullptr : static_cast<const uint8_t*>(p) + n; };
        auto code = [](uint8_t* p, size_t n) { return p == nullptr ? nullptr : p + n; };
        e.gate = byte(ep.gate, r * ep.gate_ld * size), e.residual = byte(ep.residual, r * ep.residual_ld * size);
        e.z_codes = code(ep.z_codes, r * pitch), e.z_exponents = code(ep.z_exponents, r * (pitch / kCkptBlock));
        e.gate_codes = code(ep.gate_codes, r * pitch), e.gate_exponents = code(ep.gate_exponents, r * (pitch / kCkptBlock));
        int done;
        if (tiles) {
            const GemmCall c = {a.b + r * a.k, a.a, static_cast<uint8_t*>(a.d) + r * a.m * size, dt, static_cast<int>(rows),
                                static_cast<int>(a.m), static_cast<int>(a.k), a.b_scale_inv, a.a_scale_inv, 0, a.bias,
                                static_cast<int>(a.bias_dtype), false, false, nullptr, st};
            done = dt == MSAMP_DT_F32   ? run_gemm_fused<float>(c, e)
                   : dt == MSAMP_DT_F16 ? run_gemm_fused<f16_t>(c, e)
                                        : run_gemm_fused<bf16_t>(c, e);
        } else {
            msamp_gemm_fused_args part = a;
            part.b = a.b + r * a.k, part.d = static_cast<uint8_t*>(a.d) + r * a.m * size, part.n = rows;
            done = dt == MSAMP_DT_F32   ? run_rows<float>(part, e, st)
                   : dt == MSAMP_DT_F16 ? run_rows<f16_t>(part, e, st)
                                        : run_rows<bf16_t>(part, e, st);
        }
        if (done != MSAMP_OK) return done;
    }
    return MSAMP_OK;
}
