// Activations and their slopes, 8-bit checkpoints of activations, and the epilogue that a product ends with: what the fused product
// (gemm_fused.hip, gemm_kernels.cuh) and the kernels over checkpoints (activation.hip) share.
#pragma once
#include "common.cuh"

#include <type_traits>

namespace msamp {

// ---- activations -----------------------------------------------------------------------------
// float32 throughout.  Each costs one v_exp_f32 and one v_rcp_f32 (a quarter of the rate of an addition each, within an ulp or
// two) and a handful of additions: the tile kernels evaluate 256 of them a lane with the matrix pipes idle, and the kernels over
// checkpoints have 31 (one tensor of 16 bits, to FP8) to 62 (three, with a gate) instructions a value before memory no longer bounds them.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// 1 / (1 + e^-x): 0 and 1 at the infinities
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-x)); }

// The normal distribution function as a logistic function, Phi(z) = 1 / (1 + e^(-z P(z^2))): the logarithm of Phi(z) / Phi(-z) is odd and
// grows little faster than z^2, so that one exponential and six multiply-adds hold z Phi(z) to 7e-8 for every z (P a minimax fit
// of that error; its coefficients here times -log2 e).  Evaluated in float32 Phi is within 1.6e-7 and z Phi(z) within 4e-7 and the rounding of
// that product.  Both bounds are absolute, as those of the formula with erf in float32: far on the negative side, where z Phi(z) is
// small itself, little of it is left (3e-4 of it off at -4, 0.43 at -5.5, where it is -1.0e-7).
__device__ __forceinline__ float normal_cdf(float z) {
    const float w = z * z;
    float p = fmaf(w, -5.2700861e-09f, 3.8760723e-07f);
    p = fmaf(w, p, -1.1492852e-05f);
    p = fmaf(w, p, 1.5968819e-04f);
    p = fmaf(w, p, 9.4515628e-05f);
    p = fmaf(w, p, -0.10483681f);
    p = fmaf(w, p, -2.3022082f);
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * p));
}

// gelu_tanh: (1 + tanh(u)) / 2 is the logistic function of 2 u, u = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kTanhTwice = 1.5957691216057308f, kTanhCube = 0.044715f;
// that logistic function, with z's factor in powers of two
__device__ __forceinline__ float tanh_part(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * fmaf(-kLog2e * kTanhTwice * kTanhCube * z, z, -kLog2e * kTanhTwice)));
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == MSAMP_ACT_RELU) return z <= 0.0f ? 0.0f : z;    // (a NaN stays one)
    if constexpr (ACT == MSAMP_ACT_GELU) return z * normal_cdf(z);
    if constexpr (ACT == MSAMP_ACT_GELU_TANH) return z * tanh_part(z);
    if constexpr (ACT == MSAMP_ACT_SILU) return z * logistic(z);
    return z;
}
// a smooth one is z * part: that factor and the derivative together
template <int ACT>
__device__ __forceinline__ void act_part(float z, float& part, float& slope) {
    if constexpr (ACT == MSAMP_ACT_GELU) {
        const float bell = __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e));
        part = normal_cdf(z);
        slope = fmaf(z * bell, 0.39894228040143268f, part);
    } else if constexpr (ACT == MSAMP_ACT_GELU_TANH) {
        const float zz = fminf(z * z, 1e30f);    // (finite: behind it stands a factor of 0)
        part = tanh_part(z);
        slope = fmaf(z * part * (1.0f - part), fmaf(3.0f * kTanhTwice * kTanhCube, zz, kTanhTwice), part);
    } else {
        part = logistic(z);
        slope = fmaf(z * part, 1.0f - part, part);
    }
}
// the value and the derivative
template <int ACT>
__device__ __forceinline__ void act_both(float z, float& value, float& slope) {
    if constexpr (ACT == MSAMP_ACT_RELU) {
        value = z <= 0.0f ? 0.0f : z;
        slope = z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
    } else if constexpr (ACT == MSAMP_ACT_NONE) {
        value = z, slope = 1.0f;
    } else {
        act_part<ACT>(z, value, slope);
        value *= z;
    }
}

// ---- checkpoints -----------------------------------------------------------------------------
// 32 neighbouring values of a row share a power of two 2^E, E the smallest for which none of them leaves E4M3 after a division by
// it; a lane holds eight of the 32 and four lanes side by side a block.
constexpr int kCkptBlock = MSAMP_CKPT_BLOCK;
__host__ __device__ inline int ckpt_pitch(int cols) { return (cols + kCkptBlock - 1) / kCkptBlock * kCkptBlock; }

// the largest of four lanes (0..3, 4..7, ...), in each of them
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));    // lanes 1 0 3 2
    return umax(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));    // lanes 2 3 0 1
}
// E + 127 from the bits of the largest magnitude: 448 = 1.75 * 2^8, so a mantissa above 1.75 carries into the exponent
__device__ __forceinline__ uint32_t ckpt_exponent(uint32_t top) {
    const int e = static_cast<int>((top + 0x1fffffu) >> 23) - 8;
    return static_cast<uint32_t>(e < 1 ? 1 : e);
}
// the largest magnitude of eight, NaN left out
__device__ __forceinline__ float top_of(const float* v) {
    const float a = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fabsf(v[2])), b = fmaxf(fmaxf(fabsf(v[3]), fabsf(v[4])), fabsf(v[5]));
    return fmaxf(fmaxf(a, fabsf(v[6])), fmaxf(b, fabsf(v[7])));
}
// the codes of a lane's eight values; all four lanes of the block take part.  Infinities have no code in E4M3 and become NaN, so
// that an overflow shows in what is computed from the checkpoint; the scale comes from the finite values.  (The converter
// makes 0x7f or 0xff of both.)
__device__ __forceinline__ uint2 ckpt_codes(const float* v, uint32_t& exponent) {
    uint32_t m = quad_max(__float_as_uint(top_of(v)));
    if (__builtin_expect(m >= 0x7f800000u, 0)) {    // an infinity, or eight times NaN (the four lanes of a block come here together)
        float finite[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) finite[i] = (__float_as_uint(v[i]) & 0x7fffffffu) < 0x7f800000u ? v[i] : 0.0f;
        m = quad_max(__float_as_uint(top_of(finite)));
    }
    exponent = ckpt_exponent(m);
    const float s = __uint_as_float((254u - exponent) << 23);
    return make_uint2(quant4_in_range<MSAMP_DT_E4M3>(v[0] * s, v[1] * s, v[2] * s, v[3] * s),
                      quant4_in_range<MSAMP_DT_E4M3>(v[4] * s, v[5] * s, v[6] * s, v[7] * s));
}
__device__ __forceinline__ void ckpt_values(const uint2& codes, uint32_t exponent, float* v) {
    const float s = __uint_as_float(exponent << 23);
    dequant4<MSAMP_DT_E4M3>(codes.x, v[0], v[1], v[2], v[3]);
    dequant4<MSAMP_DT_E4M3>(codes.y, v[4], v[5], v[6], v[7]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
}

// ---- eight neighbouring elements of a row -------------------------------------------------------
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Anywhere16 {
    uint4 v;
};
template <typename T>
struct Eight {
    static constexpr int kLoads = static_cast<int>(sizeof(T)) / 2;    // 16-byte accesses: one, or two of float32
    uint4 raw[kLoads];

    // VEC: the rows start on 16 bytes and hold multiples of eight elements, so all eight are there or none.  Otherwise an access is
    // aligned to an element only, which the memory takes, and the last eight of a row come one by one.
    template <bool VEC>
    __device__ __forceinline__ void load(const T* p, int valid, bool stream = false) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) raw[i] = make_uint4(0, 0, 0, 0);
        if constexpr (VEC) {
            if (valid > 0) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) raw[i] = ld16(reinterpret_cast<const uint4*>(p) + i, stream);
            }
        } else if (valid >= 8) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) raw[i] = reinterpret_cast<const Anywhere16<T>*>(p)[i].v;
        } else {
            union {
                T e[8];
                uint4 w[kLoads];
            } u;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) u.w[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < valid) u.e[i] = p[i];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) raw[i] = u.w[i];
        }
    }
    __device__ __forceinline__ void values(float* v) const {
        if constexpr (sizeof(T) == 4) {
            In16<T>::decode(raw[0], v);
            In16<T>::decode(raw[1], v + 4);
        } else {
            In16<T>::decode(raw[0], v);
        }
    }
};

__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    const v2b p = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ uint32_t two_f16(float a, float b) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const v2h p = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ void st16(void* p, const uint4& v, bool stream) {
    if (stream) {
        typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));
        const v4u_t t = {v.x, v.y, v.z, v.w};
        __builtin_nontemporal_store(t, static_cast<v4u_t*>(p));
    } else {
        *static_cast<uint4*>(p) = v;
    }
}
// rounds to T (to nearest, ties to even) and stores
template <typename T>
__device__ __forceinline__ void to_eight(const float* v, uint4* w) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
    } else if constexpr (__is_same(T, bf16_t)) {
        w[0] = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
    } else {
        w[0] = make_uint4(two_f16(v[0], v[1]), two_f16(v[2], v[3]), two_f16(v[4], v[5]), two_f16(v[6], v[7]));
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_eight(T* p, const float* v, int valid, bool stream = false) {
    uint4 w[Eight<T>::kLoads];
    to_eight<T>(v, w);
    if constexpr (VEC) {
        if (valid > 0) {
#pragma unroll
            for (int i = 0; i < Eight<T>::kLoads; ++i) st16(reinterpret_cast<uint4*>(p) + i, w[i], stream);
        }
    } else if (valid >= 8) {
#pragma unroll
        for (int i = 0; i < Eight<T>::kLoads; ++i) reinterpret_cast<Anywhere16<T>*>(p)[i].v = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < valid) Elem<T>::store(p + i, v[i]);
    }
}

// ---- the epilogue of a product --------------------------------------------------------------------
// y = act(alpha * acc + bias) * gate + residual, with the pre-activation and the gate kept as checkpoints on the way
struct Epilogue {
    const void* bias;    // nullable: [NC]
    int bias_dt;
    int act;
    const void* gate;    // nullable: rows of the output's type, gate_ld elements apart
    long long gate_ld;
    const void* residual;    // nullable, may be the output itself
    long long residual_ld;
    uint8_t* z_codes;    // nullable
    uint8_t* z_exponents;
    uint8_t* gate_codes;    // nullable
    uint8_t* gate_exponents;
    int vec;    // output, gate and residual take 16-byte accesses: whole eights, rows on 16 bytes
    // The gate and the residual are fetched past the caches: where they are larger than the memory-side cache keeps beside the rest, the
    // kernel before this one has not left them there.  us with | without, a residual, 360 MB of it beside 16384 x 4096 -> 11008 562 | 574;
    // 134 MB beside 16384 x 11008 -> 4096 471 | 480 and x 1024 -> 4096 94 | 85; 108 MB beside 12605 x 1200 -> 4304 116 | 101; 67 MB 108 | 105.
    int stream;
    int walk_plus_one;    // the 256 x 256-tile kernel: the tile walk registered for the product (QuantArgs)
};

__device__ __forceinline__ float epilogue_bias(const Epilogue& e, int c) {
    if (e.bias_dt == MSAMP_DT_F32) return static_cast<const float*>(e.bias)[c];
    if (e.bias_dt == MSAMP_DT_F16) return f16_bits_to_float(static_cast<const uint16_t*>(e.bias)[c]);
    return bf16_bits_to_float(static_cast<const uint16_t*>(e.bias)[c]);
}

// f with the activation as a constant
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
    switch (act) {
        case MSAMP_ACT_RELU: f(std::integral_constant<int, MSAMP_ACT_RELU>{}); break;
        case MSAMP_ACT_GELU: f(std::integral_constant<int, MSAMP_ACT_GELU>{}); break;
        case MSAMP_ACT_GELU_TANH: f(std::integral_constant<int, MSAMP_ACT_GELU_TANH>{}); break;
        case MSAMP_ACT_SILU: f(std::integral_constant<int, MSAMP_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, MSAMP_ACT_NONE>{}); break;
    }
}

// ---- eight neighbouring outputs of a row, whose products are v and whose bias values b -------------------------------
// The lanes of a wave that hold the eights of one block of 32 columns lie side by side, first the one of its first column, and come here
// together.  The gate and the residual are fetched before, several rows at a time.
template <typename OT>
struct EpilogueInputs {
    Eight<OT> gate, residual;
};
template <typename OT, bool VEC>
__device__ __forceinline__ void epilogue_fetch(const Epilogue& e, int row, int col, int valid, EpilogueInputs<OT>& in) {
    if (e.gate != nullptr) in.gate.template load<VEC>(static_cast<const OT*>(e.gate) + row * e.gate_ld + col, valid);
    if (e.residual != nullptr) in.residual.template load<VEC>(static_cast<const OT*>(e.residual) + row * e.residual_ld + col, valid);
}
// `valid`: how many of the eight lie inside the output (of a row past its end: none); `row_in`: the row does
template <int ACT, typename OT, bool VEC>
__device__ __forceinline__ void epilogue_eight(const Epilogue& e, OT* D, int NC, float alpha, float* v, const float* b, int row, int col, int valid,
                                               bool row_in, const EpilogueInputs<OT>& in) {
    // (the products past the last column are those of some other one)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? fmaf(v[i], alpha, b[i]) : 0.0f;
    const int pitch = ckpt_pitch(NC);
    const size_t at = static_cast<size_t>(row) * pitch + col;
    const bool keeps = row_in && col < pitch;
    auto keep = [&](uint8_t* codes, uint8_t* exponents, const float* f) __attribute__((always_inline)) {
        uint32_t x;
        const uint2 c = ckpt_codes(f, x);
        if (!keeps) return;
        *reinterpret_cast<uint2*>(codes + at) = c;
        if ((col & (kCkptBlock - 1)) == 0) exponents[at / kCkptBlock] = static_cast<uint8_t>(x);
    };
    if (e.z_codes != nullptr) keep(e.z_codes, e.z_exponents, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value<ACT>(v[i]);
    if (e.gate != nullptr) {
        float g[8];
        in.gate.values(g);    // (zeros past the last column)
        if (e.gate_codes != nullptr) keep(e.gate_codes, e.gate_exponents, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= g[i];
    }
    if (e.residual != nullptr) {
        float r[8];
        in.residual.values(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    store_eight<OT, VEC>(D + static_cast<size_t>(row) * NC + col, v, valid);
}

// The same for a wave that works through many eights, a lane's all in the same columns (e.vec).  Loads and stores are counted together and come
// back in order, so waiting for a load waits for every store before it, and what may or may not be made can't be counted: so
// each access is made by every lane, through a buffer that ends with the wave's last row, from an offset beyond any end where a lane
// has nothing there, and which of them there are is known where the code is compiled.  (With branches around them a residual of
// 16384 x 11008 bfloat16 cost 235 us beside the product, with a load every group of rows waiting for the stores of the one before.)
// Past the caches: a tile's gate, output and codes are used once, and as ordinary accesses evict the panels of the next tiles.
// Nothing else of a compute unit runs during a large tile's epilogue, so its time adds to the products'.  bfloat16 16384 x 4096 -> 11008,
// us: the product without an epilogue 495, through this one 511, SiLU 545, a residual 562, SiLU and a gate 584, and both checkpoints 686.
template <typename OT, bool GATE, bool RESIDUAL, bool KEEP, bool STREAM>
struct WaveEpilogue {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    typedef uint32_t v2u __attribute__((ext_vector_type(2)));
    static constexpr uint32_t kSize = sizeof(OT), kNowhere = 0x80000000u;
    static constexpr int kStream = 2, kLoad = STREAM ? kStream : 0;    // the nt bit
    __amdgpu_buffer_rsrc_t out, gate, residual, z_codes, z_exponents, gate_codes, gate_exponents;
    uint32_t out_at, gate_at, residual_at, codes_at, exponents_at;        // of the lane, from the wave's first row and column
    uint32_t out_row, gate_row, residual_row, codes_row, exponents_row;    // from one row to the next
    int act, cols_in;
    bool edge;

    // the buffer from `p` on, of `rows` rows `ld` bytes apart that end `before` bytes earlier than a whole row
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int rows, long long ld, long long before) {
        const long long n = rows * ld - before;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, rows > 0 && n > 0 ? static_cast<int>(n) : 0, 0x00020000);
    }
    // the wave's rows from row0 on (at most 128), its columns from col0 on (`cols` of them); the lane's eights: (lane_row, lane_col) on
    __device__ __forceinline__ WaveEpilogue(const Epilogue& e, OT* D, int NR, int NC, int row0, int col0, int cols, int lane_row, int lane_col)
        : act(e.act), cols_in(NC - col0 - lane_col), edge(col0 + cols > NC) {
        const int rows = col0 < NC ? min(NR - row0, 128) : 0, pitch = ckpt_pitch(NC);
        const bool in = lane_col < NC - col0, in_codes = lane_col < pitch - col0;
        auto lane = [&](long long ld) { return in ? (static_cast<uint32_t>(lane_row) * static_cast<uint32_t>(ld) + lane_col) * kSize : kNowhere; };
        out = buffer(D + static_cast<size_t>(row0) * NC + col0, rows, static_cast<long long>(NC) * kSize, col0 * static_cast<long long>(kSize));
        out_at = lane(NC), out_row = NC * kSize;
        if constexpr (GATE) {
            // (the last row ends with its last column, which the rows may lie far behind)
            gate = buffer(static_cast<const OT*>(e.gate) + row0 * e.gate_ld + col0, rows, e.gate_ld * kSize, (e.gate_ld - NC + col0) * kSize);
            gate_at = lane(e.gate_ld), gate_row = static_cast<uint32_t>(e.gate_ld) * kSize;
        }
        if constexpr (RESIDUAL) {
            residual = buffer(static_cast<const OT*>(e.residual) + row0 * e.residual_ld + col0, rows, e.residual_ld * kSize, (e.residual_ld - NC + col0) * kSize);
            residual_at = lane(e.residual_ld), residual_row = static_cast<uint32_t>(e.residual_ld) * kSize;
        }
        if constexpr (KEEP) {
            const size_t from = static_cast<size_t>(row0) * pitch + col0;
            codes_at = in_codes ? static_cast<uint32_t>(lane_row) * pitch + lane_col : kNowhere, codes_row = pitch;
            exponents_at = in_codes && lane_col % kCkptBlock == 0 ? (static_cast<uint32_t>(lane_row) * pitch + lane_col) / kCkptBlock : kNowhere;
            exponents_row = pitch / kCkptBlock;
            z_codes = buffer(e.z_codes + from, rows, pitch, col0);
            z_exponents = buffer(e.z_exponents + from / kCkptBlock, rows, exponents_row, col0 / kCkptBlock);
            if constexpr (GATE) {
                gate_codes = buffer(e.gate_codes + from, rows, pitch, col0);
                gate_exponents = buffer(e.gate_exponents + from / kCkptBlock, rows, exponents_row, col0 / kCkptBlock);
            }
        }
    }
    static __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, uint32_t at, Eight<OT>& x) {
#pragma unroll
        for (int i = 0; i < Eight<OT>::kLoads; ++i) {
            const v4u t = __builtin_amdgcn_raw_buffer_load_b128(from, at + 16 * i, 0, kLoad);
            x.raw[i] = make_uint4(t.x, t.y, t.z, t.w);
        }
    }
    // the gate and the residual of the lane's eight that lies `on` rows behind its first one
    __device__ __forceinline__ void fetch(int on, EpilogueInputs<OT>& in) const {
        if constexpr (GATE) load(gate, gate_at + static_cast<uint32_t>(on) * gate_row, in.gate);
        if constexpr (RESIDUAL) load(residual, residual_at + static_cast<uint32_t>(on) * residual_row, in.residual);
    }
    __device__ __forceinline__ void keep(__amdgpu_buffer_rsrc_t codes, __amdgpu_buffer_rsrc_t exponents, int on, const float* v) const {
        uint32_t x;
        const uint2 c = ckpt_codes(v, x);
        const v2u t = {c.x, c.y};
        __builtin_amdgcn_raw_buffer_store_b64(t, codes, codes_at + static_cast<uint32_t>(on) * codes_row, 0, kStream);
        __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(x), exponents, exponents_at + static_cast<uint32_t>(on) * exponents_row, 0, 0);
    }
    // The eight `on` rows behind the lane's first one, whose products are v and whose inputs are `in`; then fetches those of the one
    // `next` rows on into `in` (next < 0: none), in front of its own stores.
    template <bool REFILL>
    __device__ __forceinline__ void eight(int on, float alpha, float* v, const float* b, EpilogueInputs<OT>& in, int next) const {
        float g[8], r[8];
        if constexpr (GATE) in.gate.values(g);
        if constexpr (RESIDUAL) in.residual.values(r);
        if constexpr (REFILL) fetch(next, in);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], alpha, b[i]);
        if constexpr (KEEP) {
            if (edge) {    // the products past the last column are those of some other one
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = i < cols_in ? v[i] : 0.0f;
            }
            keep(z_codes, z_exponents, on, v);
        }
        with_activation(act, [&](auto act_c) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(act_c)::value>(v[i]);
        });
        if constexpr (GATE) {
            if constexpr (KEEP) keep(gate_codes, gate_exponents, on, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= g[i];
        }
        if constexpr (RESIDUAL) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += r[i];
        }
        uint4 w[Eight<OT>::kLoads];
        to_eight<OT>(v, w);
#pragma unroll
        for (int i = 0; i < Eight<OT>::kLoads; ++i) {
            const v4u t = {w[i].x, w[i].y, w[i].z, w[i].w};
            __builtin_amdgcn_raw_buffer_store_b128(t, out, out_at + static_cast<uint32_t>(on) * out_row + 16 * i, 0, kStream);
        }
    }
};
// true if a WaveEpilogue does what e asks for: both checkpoints or none
__device__ __forceinline__ bool wave_epilogue_takes(const Epilogue& e) {
    return e.vec && (e.gate_codes != nullptr) == (e.gate != nullptr && e.z_codes != nullptr);
}
// f with {gate, residual, checkpoints, gate and residual past the caches} as constants
template <bool MAY_STREAM = true, typename F>
__device__ __forceinline__ void with_parts(const Epilogue& e, F&& f) {
    auto with = [&](auto gate, auto residual, auto keep) __attribute__((always_inline)) {
        if constexpr (MAY_STREAM && (decltype(gate)::value || decltype(residual)::value)) {
            if (e.stream) {
                f(gate, residual, keep, std::true_type{});
                return;
            }
        }
        f(gate, residual, keep, std::false_type{});
    };
    constexpr std::true_type y{};
    constexpr std::false_type n{};
    if (e.z_codes != nullptr) {
        if (e.gate != nullptr) {
            if (e.residual != nullptr) with(y, y, y); else with(y, n, y);
        } else {
            if (e.residual != nullptr) with(n, y, y); else with(n, n, y);
        }
    } else if (e.gate != nullptr) {
        if (e.residual != nullptr) with(y, y, n); else with(y, n, n);
    } else {
        if (e.residual != nullptr) with(n, y, n); else with(n, n, n);
    }
}

}    // namespace msamp
