// 8-bit checkpoints of activations, and the gradients of an activation taken from them.
//
// All of it is bound by memory: a value costs its bytes and at most some forty instructions beside them.  A lane holds eight
// neighbouring values of a row, so that four lanes hold a block of 32, whose maximum takes two DPP moves.
#include "activation.cuh"
#include "gate.cuh"

#include <algorithm>

namespace msamp {

constexpr int kActThreads = 256;
// (a word of the workspace for every workgroup that takes maxima, 512 columns to each of them in a row)
static_assert(MSAMP_ACT_CAST_COLS == kMaxPartials * kWave * 8, "columns of a cast");

// idx / d for idx < 2^31 (d > 1): with l = ceil(log2 d) and m = floor(2^(31 + l) / d) + 1, idx * m >> (31 + l) is the quotient
struct Divisor {
    uint32_t m, d;
    int shift;
};
static Divisor divisor_of(uint32_t d) {
    int l = 1;
    while ((1ull << l) < d) ++l;
    return {static_cast<uint32_t>((1ull << (31 + l)) / d + 1), d, l - 1};
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& v) { return __umulhi(n, v.m) >> v.shift; }

// Where eight number idx of the checkpoint lies: rows of `eights` eights, `cols` values of them real.
struct Place {
    size_t row;
    int col, valid;
};
struct Rows {
    Divisor eights;
    int cols;
};
__device__ __forceinline__ Place place_of(uint32_t idx, const Rows& r) {
    const uint32_t row = quotient(idx, r.eights);
    const int col = static_cast<int>(idx - row * r.eights.d) * 8;
    return {row, col, r.cols - col};
}

// ---------------------------------------------------------------------------------------------
// One eight to a lane and no loop: the scheduler keeps enough of these short wavefronts in flight, and every value moves once.
// 16384 x 11008 bfloat16, 547 MB each way: packed in 103 us (5.3 TB/s), unpacked in 85 (6.5; a copy of that size reaches 5.1).
// 12605 x 4301 float16 out of rows 17204 bytes apart, which begin anywhere: 37 and 26 us (4.4 and 6.3 TB/s).
template <typename T, bool VEC>
__global__ __launch_bounds__(kActThreads) void ckpt_pack_kernel(const T* __restrict__ x, long long ld, Rows rows, uint32_t total,
                                                                uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
    const uint32_t idx = blockIdx.x * kActThreads + threadIdx.x;
    if (idx >= total) return;    // (whole blocks: the eights of a row are a multiple of four)
    const Place p = place_of(idx, rows);
    Eight<T> in;
    in.template load<VEC>(x + p.row * ld + p.col, p.valid);
    float v[8];
    in.values(v);
    uint32_t e;
    const uint2 c = ckpt_codes(v, e);
    *reinterpret_cast<uint2*>(codes + static_cast<size_t>(idx) * 8) = c;
    if ((idx & 3) == 0) exponents[idx >> 2] = static_cast<uint8_t>(e);
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kActThreads) void ckpt_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents,
                                                                  Rows rows, uint32_t total, T* __restrict__ out) {
    const uint32_t idx = blockIdx.x * kActThreads + threadIdx.x;
    if (idx >= total) return;
    const Place p = place_of(idx, rows);
    float v[8];
    ckpt_values(*reinterpret_cast<const uint2*>(codes + static_cast<size_t>(idx) * 8), exponents[idx >> 2], v);
    store_eight<T, VEC>(out + p.row * rows.cols + p.col, v, p.valid);
}

// ---------------------------------------------------------------------------------------------
// The gradients of y = act(z) * gate: dz = dy * gate * act'(z) and dgate = dy * act(z), with z and the gate from checkpoints.
struct GradientArgs {
    const void* dy;
    long long dy_ld;
    const uint8_t *z_codes, *z_exponents, *gate_codes, *gate_exponents;
    void* dz;       // of dy's type, or FP8 codes
    void* dgate;    // of dy's type
    int act;
    // codes: from one row to the next, and whether a lane's eight are aligned there (then those behind the last column are written too)
    int pitch, eights_aligned;
};

template <int ACT, bool GATED>
__device__ __forceinline__ void gradient_eight(const float* dy, const float* z, const float* g, float* dz, float* dg) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float value, slope;
        act_both<ACT>(z[i], value, slope);
        if constexpr (GATED) {
            dz[i] = dy[i] * slope * g[i];
            dg[i] = dy[i] * value;
        } else {
            dz[i] = dy[i] * slope;
        }
    }
}
template <bool GATED>
__device__ __forceinline__ void gradient_eight(int act, const float* dy, const float* z, const float* g, float* dz, float* dg) {
    switch (act) {
        case MSAMP_ACT_RELU: gradient_eight<MSAMP_ACT_RELU, GATED>(dy, z, g, dz, dg); break;
        case MSAMP_ACT_GELU: gradient_eight<MSAMP_ACT_GELU, GATED>(dy, z, g, dz, dg); break;
        case MSAMP_ACT_GELU_TANH: gradient_eight<MSAMP_ACT_GELU_TANH, GATED>(dy, z, g, dz, dg); break;
        case MSAMP_ACT_SILU: gradient_eight<MSAMP_ACT_SILU, GATED>(dy, z, g, dz, dg); break;
        default: gradient_eight<MSAMP_ACT_NONE, GATED>(dy, z, g, dz, dg); break;
    }
}

// A lane's eight like the kernels above.  16384 x 11008 bfloat16 with a gate and SiLU, 1.45 GB: 246 us, 5.9 TB/s.
template <typename T, bool VEC, bool GATED>
__global__ __launch_bounds__(kActThreads) void gradient_kernel(GradientArgs a, Rows rows, uint32_t total) {
    const uint32_t idx = blockIdx.x * kActThreads + threadIdx.x;
    if (idx >= total) return;
    const Place p = place_of(idx, rows);
    Eight<T> in;
    in.template load<VEC>(static_cast<const T*>(a.dy) + p.row * a.dy_ld + p.col, p.valid);
    const size_t at = static_cast<size_t>(idx) * 8;
    float dy[8], z[8], g[8], dz[8], dg[8];
    ckpt_values(*reinterpret_cast<const uint2*>(a.z_codes + at), a.z_exponents[idx >> 2], z);
    if constexpr (GATED) ckpt_values(*reinterpret_cast<const uint2*>(a.gate_codes + at), a.gate_exponents[idx >> 2], g);
    in.values(dy);
    gradient_eight<GATED>(a.act, dy, z, g, dz, dg);
    const size_t o = p.row * rows.cols + p.col;
    store_eight<T, VEC>(static_cast<T*>(a.dz) + o, dz, p.valid);
    if constexpr (GATED) store_eight<T, VEC>(static_cast<T*>(a.dgate) + o, dg, p.valid);
}

// The same with the column sums of dz (a bias gradient) beside it, dz cast on to FP8, or both.  A workgroup takes `lanes` eights of
// columns (a power of two, 4 to 64) and every gridDim.y-th group of 256 / lanes rows, so that all of them together move through the
// rows as one front; a lane keeps the sums of its eight columns in float32, and the lanes of a column add up through LDS in a fixed order:
// the same bits on every run.  gradient_finish_kernel adds up the workgroups of a strip of columns.  Their maxima go through memory as
// well: an atomic each on one word is served one after the other.
// us (all launches) with the front | with a stretch of rows to each workgroup: 16384 x 11008 bfloat16, gate, bias, to E5M2 253 | 271;
// 12605 x 4304 float16, GELU, bias, to E5M2 56 | 57, and with half as many workgroups and twice the registers 52.  Of these the slabs
// are 44 (219 MB at 5.0 TB/s, a copy's rate), the closed gate in front 2 to 4 and the sum of the slabs 4.
struct Slabs {
    int lanes_log2;
    int rows;
};

struct __attribute__((packed, aligned(1))) Anywhere8 {
    uint2 v;
};

// A smooth activation z * part(z) and its slope by table: z is a code times a power of two, four significant bits, so there are 16 of them
// in every binade.  The table has those of 2^-24 to 2^8 and of both signs, as act_part makes them; below, the two are those
// of 0 within an ulp, and beyond, they are 0 or 1 (SiLU's, the last to get there, from 2^7 on).  Five instructions and a read of the LDS
// take the place of 14 (SiLU) to 23 (GELU) a value.
constexpr int kTable = 256, kTableFrom = 103;    // of a sign; the exponent field of the first
template <bool GATED>
struct ActTable {
    static constexpr uint32_t kFloats = GATED ? 2 : 1;    // (the slope alone where no gate's gradient asks for the part)
    float at[2 * kTable * kFloats];

    static __device__ __forceinline__ bool has(int act) { return act >= MSAMP_ACT_GELU; }
    __device__ __forceinline__ void fill(int act) {
        if (!has(act)) return;
#pragma unroll
        for (int i = threadIdx.x; i < 2 * kTable; i += kActThreads) {
            const int k = i & (kTable - 1);
            float z = __uint_as_float((kTableFrom * 8u + k) << 20), part, slope;
            if (k == 0) z = 0.0f;
            if (i >= kTable) z = -z;
            switch (act) {
                case MSAMP_ACT_GELU: act_part<MSAMP_ACT_GELU>(z, part, slope); break;
                case MSAMP_ACT_GELU_TANH: act_part<MSAMP_ACT_GELU_TANH>(z, part, slope); break;
                default: act_part<MSAMP_ACT_SILU>(z, part, slope); break;
            }
            at[i * kFloats] = slope;
            if constexpr (GATED) at[i * kFloats + 1] = part;
        }
        __syncthreads();
    }
    // (of a finite z; bits 18 and 19 are 0, so the exponent and three bits behind it count steps of four)
    __device__ __forceinline__ void look(float z, float& slope, float& part) const {
        constexpr int kShift = GATED ? 17 : 18;
        constexpr uint32_t size = 4 * kFloats, from = kTableFrom * 8 * size;
        const uint32_t b = __float_as_uint(z);
        const uint32_t t = min(max((b & 0x7fffffffu) >> kShift, from), from + size * (kTable - 1)) + ((b >> 31) * (size * kTable));
        const float* p = reinterpret_cast<const float*>(reinterpret_cast<const char*>(at) + t - from);
        if constexpr (GATED) {
            const float2 both = *reinterpret_cast<const float2*>(p);
            slope = both.x, part = both.y;
        } else {
            slope = *p;
        }
    }
};
// (the table lies behind the sums: its offset less that of its first entry is a constant of the read)
template <bool GATED>
struct SlabShared {
    float sums[kActThreads][9];    // (an odd pitch: the lanes of a column lie in different banks)
    alignas(8) ActTable<GATED> table;
};
__device__ __forceinline__ bool has_nan_code(const uint2& c) {
    return ((((c.x & 0x7f7f7f7fu) + 0x01010101u) | ((c.y & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) != 0;
}

// FMT: 0 (dz in T) or an FP8 format.  TOP_ONLY: nothing is written but the maxima (the first pass while a meta's window fills).
template <typename T, bool VEC, bool GATED, int FMT, bool TOP_ONLY>
__device__ __forceinline__ float gradient_slab(const GradientArgs& a, int cols, const Slabs& s, float scale, const ActTable<GATED>& table, float* acc) {
    const int lanes = 1 << s.lanes_log2, step = kActThreads >> s.lanes_log2;
    const int seg = blockIdx.x * lanes + (threadIdx.x & (lanes - 1));
    const int col = seg * 8, valid = cols - col;
    const int pitch = ckpt_pitch(cols), eights = pitch / 8;
    const uint32_t rows = s.rows, rows_at_once = step * gridDim.y;    // (their sum passes 31 bits)
    float top = 0.0f;
    if (seg >= eights) return top;
    uint32_t row = blockIdx.y * step + (threadIdx.x >> s.lanes_log2);
    if (row >= rows) return top;
    struct Inputs {
        Eight<T> dy;
        uint2 z, gate;
        uint8_t z_exponent, gate_exponent;
    };
    const auto fetch = [&](uint32_t r, Inputs& in) {
        in.dy.template load<VEC>(static_cast<const T*>(a.dy) + r * a.dy_ld + col, valid);
        const size_t idx = static_cast<size_t>(r) * eights + seg;
        in.z = *reinterpret_cast<const uint2*>(a.z_codes + idx * 8), in.z_exponent = a.z_exponents[idx >> 2];
        if constexpr (GATED) in.gate = *reinterpret_cast<const uint2*>(a.gate_codes + idx * 8), in.gate_exponent = a.gate_exponents[idx >> 2];
    };
    const auto work = [&](uint32_t row, const Inputs& in) {
        float dy[8], z[8], g[8], dz[8], dg[8];
        ckpt_values(in.z, in.z_exponent, z);
        if constexpr (GATED) ckpt_values(in.gate, in.gate_exponent, g);
        in.dy.values(dy);
        if (table.has(a.act)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float slope, part;
                table.look(z[i], slope, part);
                dz[i] = dy[i] * slope;
                if constexpr (GATED) dz[i] *= g[i], dg[i] = dy[i] * (z[i] * part);
            }
            if (__builtin_expect(has_nan_code(in.z), 0)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) dz[i] = z[i] != z[i] ? z[i] : dz[i];
            }
        } else if (a.act == MSAMP_ACT_RELU) {
            gradient_eight<MSAMP_ACT_RELU, GATED>(dy, z, g, dz, dg);
        } else {
            gradient_eight<MSAMP_ACT_NONE, GATED>(dy, z, g, dz, dg);
        }
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i) dz[i] = i < valid ? dz[i] : 0.0f;    // (there dy is 0, but act' of a code may be NaN)
        }
        if constexpr (TOP_ONLY) {
            // (as ordered bit patterns: a NaN lies above everything)
            uint32_t m = __float_as_uint(top);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = umax(m, __float_as_uint(dz[i]) & 0x7fffffffu);
            top = __uint_as_float(m);
            return;
        }
        const size_t o = static_cast<size_t>(row) * cols + col;
        if constexpr (FMT == 0) {
            store_eight<T, VEC>(static_cast<T*>(a.dz) + o, dz, valid);
        } else {
            // (as a rule nothing leaves the format and nothing is NaN: no clamp then, and no patch)
            const float t = top_of(dz);
            bool odd = !(t * scale <= (FMT == MSAMP_DT_E4M3 ? 448.0f : 57344.0f));
#pragma unroll
            for (int i = 0; i < 8; i += 2) odd |= __builtin_isunordered(dz[i], dz[i + 1]);
            uint2 c = make_uint2(quant4_in_range<FMT>(dz[0] * scale, dz[1] * scale, dz[2] * scale, dz[3] * scale),
                                 quant4_in_range<FMT>(dz[4] * scale, dz[5] * scale, dz[6] * scale, dz[7] * scale));
            if (__builtin_expect(odd, 0)) {
                c.x = quant4<FMT>(dz[0] * scale, dz[1] * scale, dz[2] * scale, dz[3] * scale);
                c.y = quant4<FMT>(dz[4] * scale, dz[5] * scale, dz[6] * scale, dz[7] * scale);
            }
            uint8_t* q = static_cast<uint8_t*>(a.dz) + static_cast<size_t>(row) * a.pitch + col;
            if (a.eights_aligned) {
                if (col < a.pitch) *reinterpret_cast<uint2*>(q) = c;
            } else if (valid >= 8) {
                reinterpret_cast<Anywhere8*>(q)->v = c;
            } else {
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (i < valid) q[i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
            }
            top = fmaxf(top, t);    // (a NaN is skipped, as in the casts)
        }
        if constexpr (GATED) store_eight<T, VEC>(static_cast<T*>(a.dgate) + o, dg, valid);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += dz[i];
    };
    // With a gate the next row's inputs are asked for in front of this one's stores (past the end the last row's once more): 253 -> 240 us
    // at 16384 x 11008 as above.  Without one there is little to wait for, and it costs more (12605 x 4304: 52 -> 61; two rows
    // asked for together, 55 -> 57).
    if constexpr (VEC && GATED) {
        Inputs next;
        fetch(row, next);
        for (; row < rows; row += rows_at_once) {
            const Inputs in = next;
            fetch(min(row + rows_at_once, rows - 1), next);
            work(row, in);
        }
    } else {
        for (; row < rows; row += rows_at_once) {
            Inputs in;
            fetch(row, in);
            work(row, in);
        }
    }
    return top;
}

template <typename T, bool VEC, bool GATED, int FMT>
__global__ __launch_bounds__(kActThreads, VEC ? 4 : 8) void gradient_slab_kernel(GradientArgs a, int cols, Slabs s, const float* __restrict__ scale_p,
                                                                    float* scale_inv, float* __restrict__ partial,
                                                                    float* __restrict__ tops) {
    __shared__ SlabShared<GATED> lds;
    __shared__ uint32_t red[kActThreads / kWave];
    float scale = 1.0f;
    if constexpr (FMT != 0) scale = *scale_p;
    float acc[8] = {};
    lds.table.fill(a.act);
    const float top = gradient_slab<T, VEC, GATED, FMT, false>(a, cols, s, scale, lds.table, acc);
    const int lanes = 1 << s.lanes_log2;
    if (partial != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) lds.sums[threadIdx.x][i] = acc[i];
        __syncthreads();
        for (int c = threadIdx.x; c < lanes * 8; c += kActThreads) {
            float t = 0.0f;
            for (int r = c >> 3; r < kActThreads; r += lanes) t += lds.sums[r][c & 7];
            const int col = blockIdx.x * lanes * 8 + c;
            if (col < cols) partial[static_cast<size_t>(blockIdx.y) * cols + col] = t;
        }
    }
    if constexpr (FMT != 0) {
        const uint32_t m = block_max_u32(__float_as_uint(top), red);
        if (threadIdx.x == 0) {
            tops[static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x] = __uint_as_float(m);
            if (blockIdx.x == 0 && blockIdx.y == 0) *scale_inv = 1.0f / scale;
        }
    }
}

// Adds the slabs up, 16 runs of them at a time, and rounds once; workgroup 0 also folds the maxima into *amax.
template <typename OT>
__global__ __launch_bounds__(1024) void gradient_finish_kernel(const float* __restrict__ partial, OT* __restrict__ sum, int slabs, int cols,
                                                               const float* __restrict__ tops, int n_tops, float* amax) {
    __shared__ float part[16][kWave];
    __shared__ uint32_t red[16];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    if (blockIdx.x == 0 && n_tops > 0) {
        float top = 0.0f;
        for (int i = threadIdx.x; i < n_tops; i += 1024) top = fmaxf(top, tops[i]);
        const uint32_t m = block_max_u32(__float_as_uint(top), red);
        if (threadIdx.x == 0) amax_publish(amax, __uint_as_float(m));
    }
    if (sum == nullptr) return;
    const int c = blockIdx.x * kWave + lane;
    float t = 0.0f;
    if (c < cols) {
        const int per = (slabs + 15) / 16;
        const int end = min((run + 1) * per, slabs);
#pragma unroll 8
        for (int i = run * per; i < end; ++i) t += partial[static_cast<size_t>(i) * cols + c];
    }
    part[run][lane] = t;
    __syncthreads();
    if (run == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 16; ++i) t += part[i][lane];
        Elem<OT>::store(sum + c, t);
    }
}

// While the meta's window fills (else it returns at once): the maximum of |dz| and from it the scale that gradient_slab_kernel reads.
// The workgroup that draws the last ticket folds the others' maxima, as in the casts.
template <typename T, bool VEC, bool GATED>
__global__ __launch_bounds__(kActThreads) void gradient_top_kernel(GradientArgs a, int cols, Slabs s, Gate gate, Finish fin, uint32_t* ws) {
    if (gate_closed(gate)) return;
    __shared__ uint32_t red[kActThreads / kWave];
    __shared__ uint32_t s_last;
    __shared__ ActTable<GATED> table;
    table.fill(a.act);
    float none[8];
    const float top = gradient_slab<T, VEC, GATED, 0, true>(a, cols, s, 1.0f, table, none);
    uint32_t m = block_max_u32(__float_as_uint(top), red);
    const int blocks = gridDim.x * gridDim.y, block = blockIdx.y * gridDim.x + blockIdx.x;
    if (threadIdx.x == 0) {
        __hip_atomic_store(ws + kWsPartials + block, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __threadfence();    // the maximum is visible before the ticket is taken
        const uint32_t ticket = atomicAdd(ws + kWsTicket, 1u);
        s_last = ticket == static_cast<uint32_t>(blocks) - 1;
        if (s_last) ws[kWsTicket] = 0;    // ready for the next call
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    m = 0;
    for (int i = threadIdx.x; i < blocks; i += kActThreads)
        m = umax(m, __hip_atomic_load(ws + kWsPartials + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    m = block_max_u32(m, red);
    if (threadIdx.x == 0) {
        const float am = __uint_as_float(m);
        const float sc = scale_rule(am, *fin.scale, fin.fp_max, fin.margin);
        *fin.amax = am;
        *fin.scale = sc;
        *fin.scale_inv = 1.0f / sc;
    }
}

// ---- host side ---------------------------------------------------------------------------------
// calls f(first row, rows of it, total eights) for stretches of rows whose eights are counted in 31 bits
template <typename F>
static int in_stretches(long long rows, int cols, F&& f) {
    const long long eights = ckpt_pitch(cols) / 8, most = std::max(1LL, ((1LL << 31) - kActThreads) / eights);
    for (long long r = 0; r < rows; r += most) {
        const long long n = std::min(most, rows - r);
        const int rc = f(r, n, static_cast<uint32_t>(n * eights));
        if (rc != MSAMP_OK) return rc;
    }
    return MSAMP_OK;
}

template <typename T>
static int launch_pack(const T* x, long long rows, int cols, long long ld, uint8_t* codes, uint8_t* exponents, hipStream_t st) {
    const bool vec = cols % 8 == 0 && ld * sizeof(T) % 16 == 0 && aligned(x, 16);
    const size_t pitch = ckpt_pitch(cols);
    const Rows shape = {divisor_of(static_cast<uint32_t>(pitch / 8)), cols};
    return in_stretches(rows, cols, [&](long long r, long long, uint32_t total) {
        const dim3 grid((total + kActThreads - 1) / kActThreads);
        const auto kern = vec ? ckpt_pack_kernel<T, true> : ckpt_pack_kernel<T, false>;
        hipLaunchKernelGGL(kern, grid, dim3(kActThreads), 0, st, x + r * ld, ld, shape, total, codes + r * pitch, exponents + r * (pitch / kCkptBlock));
        MSAMP_CHECK_LAUNCH("ckpt_pack_kernel");
        return static_cast<int>(MSAMP_OK);
    });
}

template <typename T>
static int launch_unpack(const uint8_t* codes, const uint8_t* exponents, long long rows, int cols, T* out, hipStream_t st) {
    const bool vec = cols % 8 == 0 && aligned(out, 16);
    const size_t pitch = ckpt_pitch(cols);
    const Rows shape = {divisor_of(static_cast<uint32_t>(pitch / 8)), cols};
    return in_stretches(rows, cols, [&](long long r, long long, uint32_t total) {
        const dim3 grid((total + kActThreads - 1) / kActThreads);
        const auto kern = vec ? ckpt_unpack_kernel<T, true> : ckpt_unpack_kernel<T, false>;
        hipLaunchKernelGGL(kern, grid, dim3(kActThreads), 0, st, codes + r * pitch, exponents + r * (pitch / kCkptBlock), shape, total, out + r * cols);
        MSAMP_CHECK_LAUNCH("ckpt_unpack_kernel");
        return static_cast<int>(MSAMP_OK);
    });
}

// Workgroups of the kernels over slabs.  Whole eights: all at work at once, four to a compute unit, whose registers hold more loads on their
// way than eight of them (12605 x 4304 52 us | 56, 16384 x 11008 with gate and bias 290 | 306).  Eights that begin anywhere are loaded
// piece by piece where a row ends, which needs the wavefronts: two rounds of eight (12605 x 4301 62 us; one round 66, one of four 78).
static int slab_workgroups(bool vec) { return cu_count() * (vec ? 4 : 16); }
// As many lanes to a row as its eights fill, at most a wavefront, and about `most` workgroups.
struct SlabGrid {
    Slabs s;
    int strips, slabs;
};
static SlabGrid slab_grid(int rows, int cols, int most) {
    const int eights = ckpt_pitch(cols) / 8;
    int log2 = 2;
    while (log2 < 6 && (1 << log2) < eights) ++log2;
    const int lanes = 1 << log2, at_once = kActThreads / lanes, strips = (eights + lanes - 1) / lanes;
    return {{log2, rows}, strips, std::min(std::max(1, most / strips), (rows - 1) / at_once + 1)};
}

template <typename T, bool VEC, bool GATED>
static int launch_gradient(const msamp_activation_backward_args& a, const GradientArgs& g, hipStream_t st) {
    const int rows = static_cast<int>(a.rows), cols = static_cast<int>(a.cols);
    const int fmt = static_cast<int>(a.dz_type);
    if (!is_fp8(fmt) && a.bias_sum == nullptr) {
        const size_t pitch = ckpt_pitch(cols);
        const Rows shape = {divisor_of(static_cast<uint32_t>(pitch / 8)), cols};
        return in_stretches(rows, cols, [&](long long r, long long, uint32_t total) {
            GradientArgs p = g;
            p.dy = static_cast<const T*>(g.dy) + r * g.dy_ld;
            p.z_codes = g.z_codes + r * pitch, p.z_exponents = g.z_exponents + r * (pitch / kCkptBlock);
            p.dz = static_cast<T*>(g.dz) + r * cols;
            if constexpr (GATED) {
                p.gate_codes = g.gate_codes + r * pitch, p.gate_exponents = g.gate_exponents + r * (pitch / kCkptBlock);
                p.dgate = static_cast<T*>(g.dgate) + r * cols;
            }
            hipLaunchKernelGGL((gradient_kernel<T, VEC, GATED>), dim3((total + kActThreads - 1) / kActThreads), dim3(kActThreads), 0, st, p, shape, total);
            MSAMP_CHECK_LAUNCH("gradient_kernel");
            return static_cast<int>(MSAMP_OK);
        });
    }
    const SlabGrid sg = slab_grid(rows, cols, slab_workgroups(VEC));
    const dim3 grid(sg.strips, sg.slabs);
    float* partial = a.bias_sum != nullptr ? static_cast<float*>(a.scratch) : nullptr;
    float* tops = static_cast<float*>(a.scratch) + (a.bias_sum != nullptr ? static_cast<size_t>(sg.slabs) * cols : 0);
    if (is_fp8(fmt)) {
        const Gate gate = {a.counter, static_cast<int>(a.window)};
        const Finish fin = {a.amax, a.scale, a.scale_inv, fp8_max(fmt), 0, 0};
        // (As a rule the gate is closed and its workgroups return at once: few of them.  While the window fills they read everything once
        // more, slowly: bfloat16, GELU, bias, to E5M2 12605 x 4304 120 us instead of 46, 16384 x 11008 436 instead of 144.)
        const SlabGrid few = slab_grid(rows, cols, std::min(cu_count(), kMaxPartials));
        hipLaunchKernelGGL((gradient_top_kernel<T, VEC, GATED>), dim3(few.strips, few.slabs), dim3(kActThreads), 0, st, g, cols, few.s, gate, fin,
                           static_cast<uint32_t*>(a.workspace));
        MSAMP_CHECK_LAUNCH("gradient_top_kernel");
    }
    const auto kern = fmt == MSAMP_DT_E5M2   ? gradient_slab_kernel<T, VEC, GATED, MSAMP_DT_E5M2>
                      : fmt == MSAMP_DT_E4M3 ? gradient_slab_kernel<T, VEC, GATED, MSAMP_DT_E4M3>
                                             : gradient_slab_kernel<T, VEC, GATED, 0>;
    hipLaunchKernelGGL(kern, grid, dim3(kActThreads), 0, st, g, cols, sg.s, static_cast<const float*>(a.scale), a.scale_inv, partial, tops);
    MSAMP_CHECK_LAUNCH("gradient_slab_kernel");
    const int n_tops = is_fp8(fmt) ? sg.strips * sg.slabs : 0;
    const dim3 fgrid(a.bias_sum != nullptr ? (cols + kWave - 1) / kWave : 1);
#define FINISH(OT) \
    hipLaunchKernelGGL(gradient_finish_kernel<OT>, fgrid, dim3(1024), 0, st, static_cast<const float*>(partial), static_cast<OT*>(a.bias_sum), sg.slabs, cols, static_cast<const float*>(tops), n_tops, a.amax)
    if (a.bias_sum_dtype == MSAMP_DT_F16) FINISH(f16_t);
    else if (a.bias_sum_dtype == MSAMP_DT_BF16) FINISH(bf16_t);
    else FINISH(float);
#undef FINISH
    MSAMP_CHECK_LAUNCH("gradient_finish_kernel");
    return MSAMP_OK;
}

template <typename T>
static int launch_gradient_of(const msamp_activation_backward_args& a, const GradientArgs& g, hipStream_t st) {
    const bool gated = a.gate_codes != nullptr;
    const bool vec = a.cols % 8 == 0 && a.dy_stride * sizeof(T) % 16 == 0 && aligned(a.dy, 16) &&
                     (is_fp8(static_cast<int>(a.dz_type)) || aligned(a.dz, 16)) && (!gated || aligned(a.dgate, 16));
    if (gated) return vec ? launch_gradient<T, true, true>(a, g, st) : launch_gradient<T, false, true>(a, g, st);
    return vec ? launch_gradient<T, true, false>(a, g, st) : launch_gradient<T, false, false>(a, g, st);
}

}    // namespace msamp

using namespace msamp;

extern "C" {

int msamp_checkpoint_pack(const void* x, int dtype, long long rows, long long cols, long long row_stride, uint8_t* codes, uint8_t* exponents,
                          msamp_stream_t stream) {
    MSAMP_REQUIRE(is_hp(dtype), MSAMP_ERR_DTYPE, "msamp_checkpoint_pack: dtype %d", dtype);
    MSAMP_REQUIRE(rows >= 0 && cols >= 0 && cols <= MSAMP_CKPT_COLS && (rows <= 1 || row_stride >= cols), MSAMP_ERR_SHAPE,
                  "msamp_checkpoint_pack: %lld x %lld, rows %lld apart", rows, cols, row_stride);
    if (rows == 0 || cols == 0) return MSAMP_OK;
    MSAMP_REQUIRE(x && codes && exponents, MSAMP_ERR_NULL, "msamp_checkpoint_pack: null pointer");
    MSAMP_REQUIRE(aligned(codes, 16), MSAMP_ERR_ALIGNMENT, "msamp_checkpoint_pack: codes must be 16-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int width = static_cast<int>(cols);
    if (dtype == MSAMP_DT_F32) return launch_pack(static_cast<const float*>(x), rows, width, row_stride, codes, exponents, st);
    if (dtype == MSAMP_DT_F16) return launch_pack(static_cast<const f16_t*>(x), rows, width, row_stride, codes, exponents, st);
    return launch_pack(static_cast<const bf16_t*>(x), rows, width, row_stride, codes, exponents, st);
}

int msamp_checkpoint_unpack(const uint8_t* codes, const uint8_t* exponents, long long rows, long long cols, void* out, int dtype,
                            msamp_stream_t stream) {
    MSAMP_REQUIRE(is_hp(dtype), MSAMP_ERR_DTYPE, "msamp_checkpoint_unpack: dtype %d", dtype);
    MSAMP_REQUIRE(rows >= 0 && cols >= 0 && cols <= MSAMP_CKPT_COLS, MSAMP_ERR_SHAPE, "msamp_checkpoint_unpack: %lld x %lld", rows, cols);
    if (rows == 0 || cols == 0) return MSAMP_OK;
    MSAMP_REQUIRE(codes && exponents && out, MSAMP_ERR_NULL, "msamp_checkpoint_unpack: null pointer");
    MSAMP_REQUIRE(aligned(codes, 16), MSAMP_ERR_ALIGNMENT, "msamp_checkpoint_unpack: codes must be 16-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int width = static_cast<int>(cols);
    if (dtype == MSAMP_DT_F32) return launch_unpack(codes, exponents, rows, width, static_cast<float*>(out), st);
    if (dtype == MSAMP_DT_F16) return launch_unpack(codes, exponents, rows, width, static_cast<f16_t*>(out), st);
    return launch_unpack(codes, exponents, rows, width, static_cast<bf16_t*>(out), st);
}

int msamp_activation_backward_scratch(long long rows, long long cols, int want_bias, int fp8, size_t* bytes) {
    MSAMP_REQUIRE(rows > 0 && cols > 0 && rows <= 0x7fffffffLL && cols <= MSAMP_CKPT_COLS, MSAMP_ERR_SHAPE,
                  "msamp_activation_backward_scratch: %lld x %lld", rows, cols);
    MSAMP_REQUIRE(bytes != nullptr, MSAMP_ERR_NULL, "msamp_activation_backward_scratch: null pointer");
    MSAMP_REQUIRE(!fp8 || cols <= MSAMP_ACT_CAST_COLS, MSAMP_ERR_SHAPE, "msamp_activation_backward_scratch: a cast of %lld columns", cols);
    const SlabGrid sg = slab_grid(static_cast<int>(rows), static_cast<int>(cols), slab_workgroups(false));    // (the larger of the two)
    *bytes = 4 * ((want_bias ? static_cast<size_t>(sg.slabs) * cols : 0) + (fp8 ? static_cast<size_t>(sg.slabs) * sg.strips : 0));
    return MSAMP_OK;
}

int msamp_activation_backward(const msamp_activation_backward_args* args, msamp_stream_t stream) {
    MSAMP_REQUIRE(args != nullptr, MSAMP_ERR_NULL, "msamp_activation_backward: null pointer");
    const msamp_activation_backward_args& a = *args;
    const bool gated = a.gate_codes != nullptr, fp8 = is_fp8(static_cast<int>(a.dz_type));
    MSAMP_REQUIRE(is_hp(static_cast<int>(a.dy_dtype)) && (fp8 || a.dz_type == a.dy_dtype), MSAMP_ERR_DTYPE,
                  "msamp_activation_backward: dy type %d, dz type %d", static_cast<int>(a.dy_dtype), static_cast<int>(a.dz_type));
    MSAMP_REQUIRE(a.bias_sum == nullptr || is_hp(static_cast<int>(a.bias_sum_dtype)), MSAMP_ERR_DTYPE,
                  "msamp_activation_backward: bias_sum_dtype %d", static_cast<int>(a.bias_sum_dtype));
    MSAMP_REQUIRE(a.activation >= MSAMP_ACT_NONE && a.activation <= MSAMP_ACT_SILU, MSAMP_ERR_DTYPE,
                  "msamp_activation_backward: activation %d", static_cast<int>(a.activation));
    MSAMP_REQUIRE(a.rows > 0 && a.cols > 0 && a.rows <= 0x7fffffffLL && a.cols <= MSAMP_CKPT_COLS && (a.rows == 1 || a.dy_stride >= a.cols),
                  MSAMP_ERR_SHAPE, "msamp_activation_backward: %lld x %lld, rows of dy %lld apart", static_cast<long long>(a.rows),
                  static_cast<long long>(a.cols), static_cast<long long>(a.dy_stride));
    MSAMP_REQUIRE(a.dy && a.z_codes && a.z_exponents && a.dz && (!gated || (a.gate_exponents && a.dgate)), MSAMP_ERR_NULL,
                  "msamp_activation_backward: null pointer");
    MSAMP_REQUIRE(!fp8 || a.dz_pitch == a.cols || (a.dz_pitch == (a.cols + 15) / 16 * 16 && aligned(a.dz, 16)), MSAMP_ERR_SHAPE,
                  "msamp_activation_backward: codes in rows of %lld", static_cast<long long>(a.dz_pitch));
    MSAMP_REQUIRE(!fp8 || (a.scale && a.amax && a.scale_inv && a.counter), MSAMP_ERR_NULL, "msamp_activation_backward: null pointer in the meta");
    MSAMP_REQUIRE(!fp8 || a.workspace, MSAMP_ERR_WORKSPACE, "msamp_activation_backward: workspace required");
    MSAMP_REQUIRE(aligned(a.z_codes, 16) && aligned(a.gate_codes, 16), MSAMP_ERR_ALIGNMENT,
                  "msamp_activation_backward: codes must be 16-byte aligned");
    if (fp8 || a.bias_sum != nullptr) {
        size_t need = 0;
        const int rc = msamp_activation_backward_scratch(a.rows, a.cols, a.bias_sum != nullptr, fp8, &need);
        if (rc != MSAMP_OK) return rc;
        MSAMP_REQUIRE(a.scratch != nullptr && static_cast<size_t>(a.scratch_bytes) >= need && aligned(a.scratch, 4), MSAMP_ERR_WORKSPACE,
                      "msamp_activation_backward: scratch of %zu bytes required", need);
    }
    const GradientArgs g = {a.dy, a.dy_stride, a.z_codes, a.z_exponents, a.gate_codes, a.gate_exponents, a.dz, a.dgate, static_cast<int>(a.activation),
                            static_cast<int>(a.dz_pitch), a.dz_pitch % 8 == 0 && aligned(a.dz, 8)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.dy_dtype == MSAMP_DT_F32) return launch_gradient_of<float>(a, g, st);
    if (a.dy_dtype == MSAMP_DT_F16) return launch_gradient_of<f16_t>(a, g, st);
    return launch_gradient_of<bf16_t>(a, g, st);
}

}    // extern "C"
