// experts_formats.hpp -- from a laid out unit's bytes (experts.hpp) to the B operands of v_mfma_f32_32x32x16_f16: exact
// integers in fp16 (FP16: the weights themselves), and the scales that the fp32 partial sums take.
//
// ExpertFmt<FMT>: load(q, unit, stage) a lane's bytes of a stage of four steps (64 k), in kLoads loads, load(s, unit) those of
// the unit's scales; operand<J, S>(q, s, b) the eight weights of step S of stage J, as four pairs.  kScaled says how scales are
// applied: kNoScale not at all; kPerStep and kPerBlock the partial sum of a step (16 k) or of a block of two times part_scale<I>() (I: the
// unit's step or block).  Q4_K's minimums meet the activations' sums over 32, which are staged times 2^-6, once per unit:
// min_operand(), min_scale().
//
// Scales multiply a partial sum instead of the weights because d q has 19 bits, fp16 11.  Other forms that fit: Q4_K's 6-bit
// scale times 4-bit code (10 bits) in the operand, d per unit, half the scalings: its 64 registers of unit sums spill, 4096
// tokens' SwiGLU 630 us against 591 as Q4_0 does it; Q6_K's scale times code (12 bits) as an operand's nearest half and its rest
// in a third MFMA, no scalings before the unit's end: 856 us against 790, the MFMAs' power counts; Q4_K's codes as fp16's
// smallest numbers, masked alone: 555 us against 581, but the products lose bits, errors of 1e-5 instead of 3e-7.
#pragma once

#include "experts.hpp"

namespace cri {
namespace dev {

enum : int { kNoScale = 0, kPerStep = 1, kPerBlock = 2 };

typedef _Float16 eh2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t e_splat(float v) {  // v in both halves
    const uint16_t h = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
    return static_cast<uint32_t>(h) | (static_cast<uint32_t>(h) << 16);
}
__device__ __forceinline__ uint32_t e_fma(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(eh2, a), __builtin_bit_cast(eh2, b),
                                                                  __builtin_bit_cast(eh2, c)));
}
__device__ __forceinline__ uint32_t e_add(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(eh2, a) + __builtin_bit_cast(eh2, b));
}
// (v & m) | o as one v_and_or_b32: the constants are kept from the compiler, which would take two instructions with literals.
// (Not as an instruction in asm: the compiler does not see that one write registers that an MFMA is still to write.)
__device__ __forceinline__ uint32_t e_and_or(uint32_t v, uint32_t m, uint32_t o) {
    asm("" : "+s"(m));
    asm("" : "+v"(o));
    return (v & m) | o;
}
constexpr uint32_t kTop = 0x64006400u;     // 1024 in both halves
constexpr uint32_t kTenth = 0x2C002C00u;   // 1/16 in both halves

// 16 bytes at a wave-uniform address and the lane's offset (one SGPR pair, one VGPR)
__device__ __forceinline__ u32x4 e_load16(const uint8_t* p, uint32_t off) { return *reinterpret_cast<const u32x4*>(p + off); }
__device__ __forceinline__ float e_half(uint32_t w, bool high) { return high ? h_hi(w) : h_lo(w); }

// The compiler waits for v's loads here.
__device__ __forceinline__ void e_settle(u32x4& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void e_settle(uint32_t& v) { asm volatile("" : "+v"(v)); }

template <int FMT>
struct ExpertFmt;

// nibbles of a step to four pairs: t[0], t[2] are 1024 + q, t[1], t[3] are 1024 + 16 q
__device__ __forceinline__ void e_nibbles(uint32_t x, uint32_t (&t)[4]) {
    const uint32_t y = x >> 8;
    t[0] = e_and_or(x, 0x000F000Fu, kTop);
    t[1] = e_and_or(x, 0x00F000F0u, kTop);
    t[2] = e_and_or(y, 0x000F000Fu, kTop);
    t[3] = e_and_or(y, 0x00F000F0u, kTop);
}

struct NibbleQuant {
    u32x4 q;
    __device__ __forceinline__ void settle() { e_settle(q); }
};
__device__ __forceinline__ uint32_t e_at(const u32x4& v, int i) { return v[i]; }

template <>
struct ExpertFmt<kFmtQ4_0> {
    static constexpr int kScaled = kPerBlock, kLoads = 1;
    typedef NibbleQuant Quant;
    struct Scale {
        u32x4 d;
    };
    static __device__ __forceinline__ void load(Quant& q, const uint8_t* unit, int stage, uint32_t lane) {
        q.q = e_load16(unit + 1024 * stage, 16 * lane);
    }
    static __device__ __forceinline__ void load(Scale& s, const uint8_t* unit, uint32_t lane) {
        s.d = e_load16(unit + 4096, 16 * (lane & 31));
    }
    template <int J, int S>
    static __device__ __forceinline__ void operand(const Quant& q, const Scale&, uint32_t (&b)[4]) {
        uint32_t t[4];
        e_nibbles(e_at(q.q, S), t);
        const uint32_t low = e_splat(-1032.0f), high = e_splat(-72.0f);  // -(1024 + 8), -(1024 / 16 + 8)
        b[0] = e_add(t[0], low);
        b[1] = e_fma(t[1], kTenth, high);
        b[2] = e_add(t[2], low);
        b[3] = e_fma(t[3], kTenth, high);
    }
    template <int I>
    static __device__ __forceinline__ float part_scale(const Scale& s) {
        return e_half(s.d[I >> 1], I & 1);
    }
};

template <>
struct ExpertFmt<kFmtQ8_0> {
    static constexpr int kScaled = kPerBlock, kLoads = 2;
    struct Quant {
        u32x4 q[2];
        __device__ __forceinline__ void settle() { e_settle(q[0]), e_settle(q[1]); }
    };
    struct Scale {
        u32x4 d;
    };
    static __device__ __forceinline__ void load(Quant& q, const uint8_t* unit, int stage, uint32_t lane) {
        q.q[0] = e_load16(unit + 2048 * stage, 16 * lane);
        q.q[1] = e_load16(unit + 2048 * stage + 1024, 16 * lane);
    }
    static __device__ __forceinline__ void load(Scale& s, const uint8_t* unit, uint32_t lane) {
        s.d = e_load16(unit + 8192, 16 * (lane & 31));
    }
    template <int J, int S>
    static __device__ __forceinline__ void operand(const Quant& q, const Scale&, uint32_t (&b)[4]) {
        const uint32_t zero = e_splat(-1152.0f);  // -(1024 + 128)
        const uint32_t x = q.q[S >> 1][2 * (S & 1)], y = q.q[S >> 1][2 * (S & 1) + 1];
        b[0] = e_add(e_and_or(x, 0x00FF00FFu, kTop), zero);
        b[1] = e_add(e_and_or(x >> 8, 0x00FF00FFu, kTop), zero);
        b[2] = e_add(e_and_or(y, 0x00FF00FFu, kTop), zero);
        b[3] = e_add(e_and_or(y >> 8, 0x00FF00FFu, kTop), zero);
    }
    template <int I>
    static __device__ __forceinline__ float part_scale(const Scale& s) {
        return e_half(s.d[I >> 1], I & 1);
    }
};

// w's bits from position `from` to position `to`
__device__ __forceinline__ uint32_t e_move(uint32_t w, int from, int to) { return from >= to ? w >> (from - to) : w << (to - from); }

template <>
struct ExpertFmt<kFmtQ5_0> {
    static constexpr int kScaled = kPerBlock, kLoads = 2;
    struct Quant {
        u32x4 q;
        uint32_t h;
        __device__ __forceinline__ void settle() { e_settle(q), e_settle(h); }
    };
    struct Scale {
        u32x4 d;
    };
    static __device__ __forceinline__ void load(Quant& q, const uint8_t* unit, int stage, uint32_t lane) {
        q.q = e_load16(unit + 1024 * stage, 16 * lane);
        q.h = *reinterpret_cast<const uint32_t*>(unit + (4096 + 4 * stage) + 16 * lane);
    }
    static __device__ __forceinline__ void load(Scale& s, const uint8_t* unit, uint32_t lane) {
        s.d = e_load16(unit + 5120, 16 * (lane & 31));
    }
    template <int J, int S>
    static __device__ __forceinline__ void operand(const Quant& q, const Scale&, uint32_t (&b)[4]) {
        uint32_t t[4];
        e_nibbles(e_at(q.q, S), t);
        const uint32_t low = e_splat(-1040.0f), high = e_splat(-80.0f);  // -(1024 + 16), -(1024 / 16 + 16)
        b[0] = e_add(e_and_or(e_move(q.h, 4 * S, 4), 0x00100010u, t[0]), low);
        b[1] = e_fma(e_and_or(e_move(q.h, 4 * S + 1, 8), 0x01000100u, t[1]), kTenth, high);
        b[2] = e_add(e_and_or(e_move(q.h, 4 * S + 2, 4), 0x00100010u, t[2]), low);
        b[3] = e_fma(e_and_or(e_move(q.h, 4 * S + 3, 8), 0x01000100u, t[3]), kTenth, high);
    }
    template <int I>
    static __device__ __forceinline__ float part_scale(const Scale& s) {
        return e_half(s.d[I >> 1], I & 1);
    }
};

template <>
struct ExpertFmt<kFmtQ6_K> {
    static constexpr int kScaled = kPerStep, kLoads = 2;
    struct Quant {
        u32x4 q;
        uint32_t h[2];
        __device__ __forceinline__ void settle() { e_settle(q), e_settle(h[0]), e_settle(h[1]); }
    };
    struct Scale {
        u32x4 sc;
        uint32_t d;
    };
    static __device__ __forceinline__ void load(Quant& q, const uint8_t* unit, int stage, uint32_t lane) {
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        q.q = e_load16(unit + 1024 * stage, 16 * lane);
        const u2 h = *reinterpret_cast<const u2*>(unit + (4096 + 1024 * (stage >> 1) + 8 * (stage & 1)) + 16 * lane);
        q.h[0] = h.x;
        q.h[1] = h.y;
    }
    static __device__ __forceinline__ void load(Scale& s, const uint8_t* unit, uint32_t lane) {
        s.sc = e_load16(unit + 6144, 16 * (lane & 31));
        s.d = *reinterpret_cast<const uint16_t*>(unit + 6656 + 2 * (lane & 31));
    }
    template <int J, int S>
    static __device__ __forceinline__ void operand(const Quant& q, const Scale&, uint32_t (&b)[4]) {
        uint32_t t[4];
        e_nibbles(e_at(q.q, S), t);
        const uint32_t h = q.h[S >> 1];
        constexpr int o = 8 * (S & 1);
        const uint32_t low = e_splat(-1056.0f), high = e_splat(-96.0f);  // -(1024 + 32), -(1024 / 16 + 32)
        b[0] = e_add(e_and_or(e_move(h, o, 4), 0x00300030u, t[0]), low);
        b[1] = e_fma(e_and_or(e_move(h, o + 2, 8), 0x03000300u, t[1]), kTenth, high);
        b[2] = e_add(e_and_or(e_move(h, o + 4, 4), 0x00300030u, t[2]), low);
        b[3] = e_fma(e_and_or(e_move(h, o + 6, 8), 0x03000300u, t[3]), kTenth, high);
    }
    template <int I>
    static __device__ __forceinline__ float part_scale(const Scale& s) {
        return h_lo(s.d) * sbyte(s.sc[I >> 2], I & 3);  // 19 bits: exact
    }
};

template <>
struct ExpertFmt<kFmtQ4_K> {
    static constexpr int kScaled = kPerBlock, kLoads = 1;
    typedef NibbleQuant Quant;
    struct Scale {
        u32x4 s;  // sc, mn
        uint32_t d;
    };
    static __device__ __forceinline__ void load(Quant& q, const uint8_t* unit, int stage, uint32_t lane) {
        q.q = e_load16(unit + 1024 * stage, 16 * lane);
    }
    static __device__ __forceinline__ void load(Scale& s, const uint8_t* unit, uint32_t lane) {
        s.s = e_load16(unit + 4096, 16 * (lane & 31));
        s.d = *reinterpret_cast<const uint32_t*>(unit + 4608 + 4 * (lane & 31));
    }
    template <int J, int S>
    static __device__ __forceinline__ void operand(const Quant& q, const Scale&, uint32_t (&b)[4]) {
        uint32_t t[4];
        e_nibbles(e_at(q.q, S), t);
        const uint32_t low = e_splat(-1024.0f), high = e_splat(-64.0f);
        b[0] = e_add(t[0], low);
        b[1] = e_fma(t[1], kTenth, high);
        b[2] = e_add(t[2], low);
        b[3] = e_fma(t[3], kTenth, high);
    }
    template <int I>
    static __device__ __forceinline__ float part_scale(const Scale& s) {
        return h_lo(s.d) * ubyte(I < 4 ? s.s.x : s.s.y, I & 3);  // 17 bits: exact
    }
    // the unit's minimums as an operand that meets the activations' sums, and what their product is multiplied by
    static __device__ __forceinline__ void min_operand(const Scale& s, uint32_t (&b)[4]) {
        const uint32_t z = e_splat(-1024.0f);
        b[0] = e_add(__builtin_amdgcn_perm(kTop, s.s.z, 0x05010500u), z);
        b[1] = e_add(__builtin_amdgcn_perm(kTop, s.s.z, 0x05030502u), z);
        b[2] = e_add(__builtin_amdgcn_perm(kTop, s.s.w, 0x05010500u), z);
        b[3] = e_add(__builtin_amdgcn_perm(kTop, s.s.w, 0x05030502u), z);
    }
    static __device__ __forceinline__ float min_scale(const Scale& s) { return -64.0f * h_hi(s.d); }
};

template <>
struct ExpertFmt<kFmtF16> {
    static constexpr int kScaled = kNoScale, kLoads = 4;
    struct Quant {
        u32x4 q[4];
        __device__ __forceinline__ void settle() { e_settle(q[0]), e_settle(q[1]), e_settle(q[2]), e_settle(q[3]); }
    };
    struct Scale {};
    static __device__ __forceinline__ void load(Quant& q, const uint8_t* unit, int stage, uint32_t lane) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q.q[i] = e_load16(unit + 4096 * stage + 1024 * i, 16 * lane);
    }
    static __device__ __forceinline__ void load(Scale&, const uint8_t*, uint32_t) {}
    template <int J, int S>
    static __device__ __forceinline__ void operand(const Quant& q, const Scale&, uint32_t (&b)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = q.q[S][i];
    }
};

}  // namespace dev
}  // namespace cri
