// Shared by the rotary, paged-cache and paged-attention kernels: typed loads and
// stores, the device form of the cache's description, and launches that may overlap
// the end of the kernel before them.
#pragma once

#include <cuda_fp8.h>

#include "epq_common.cuh"
#include "epq_paged.h"

namespace epq {
namespace paged {

// What a kernel found wrong, kept in one word a file until epq_device_error reads it.
constexpr int kBadPosition = 1;   // a position, length or sequence outside the cache or the rotary table
constexpr int kBadPage = 2;       // a page outside the pool

// Lets the next kernel of the stream start its launch, and waits for the one before.
__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const char* what,
           Args... args) {
    if (smem > 48 * 1024) {
        const int rc = set_smem_limit(reinterpret_cast<const void*>(kern), (int)smem, what);
        if (rc != EPQ_OK) return rc;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
    return check_launch(what);
}

// float <-> T, rounded to nearest even.
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values to one word and back; conversions go two at a time.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// V consecutive values; the address is aligned to their size (at most 16 bytes a load).
template <int kBytes> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };
template <> struct Word<32> { struct type { uint4 a, b; }; };

template <typename T, int V>
__device__ __forceinline__ void load_v(float (&f)[V], const T* p) {
    using W = typename Word<V * (int)sizeof(T)>::type;
    if constexpr (sizeof(T) == 2 && V > 1) {
        union { W w; uint32_t u[V / 2]; } u;
        u.w = *reinterpret_cast<const W*>(p);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 t = unpack2<T>(u.u[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    } else {
        union { W w; T t[V]; } u;
        u.w = *reinterpret_cast<const W*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f<T>(u.t[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&f)[V]) {
    using W = typename Word<V * (int)sizeof(T)>::type;
    if constexpr (sizeof(T) == 2 && V > 1) {
        union { W w; uint32_t u[V / 2]; } u;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) u.u[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        *reinterpret_cast<W*>(p) = u.w;
    } else {
        union { W w; T t[V]; } u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.t[i] = from_f<T>(f[i]);
        *reinterpret_cast<W*>(p) = u.w;
    }
}

// Eight values of a row as they lie in memory.
template <typename T> struct Eight {                    // 16-bit types: two a word
    uint32_t w[4];
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0u; }
    __device__ __forceinline__ void load(const T* p, bool aligned) {
        if (aligned) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void store(T* p, bool aligned) const {
        if (aligned) {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = unpack2<T>(w[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ Eight from_lane(int lane) const {
        Eight o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o.w[i] = __shfl_sync(0xffffffffu, w[i], lane);
        return o;
    }
    // max |x| over the kLanes lanes of a row, compared as integers so that a NaN is the largest
    template <int kLanes> __device__ __forceinline__ float largest() const {
        uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                              __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        m = max(m & 0xffffu, m >> 16);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        return unpack2<T>(m).x;
    }
};
template <> struct Eight<float> {
    float w[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0.f;
    }
    __device__ __forceinline__ void load(const float* p, bool aligned) {
        if (aligned) {
            load_v<float, 8>(w, p);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(float* p, bool aligned) const {
        if (aligned) {
            store_v<float, 8>(p, w);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = w[i];
        }
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = w[i];
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = f[i];
    }
    __device__ __forceinline__ Eight from_lane(int lane) const {
        Eight o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o.w[i] = __shfl_sync(0xffffffffu, w[i], lane);
        return o;
    }
    template <int kLanes> __device__ __forceinline__ float largest() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(w[i]) & 0x7fffffffu);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        return __uint_as_float(m);
    }
};

// One pair turned by (c, s): every product rounded, as elementwise float32 code does
// it, so results equal x1 * c - x2 * s written with tensors bit for bit.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a, y = b;
    a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    b = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
}

// Two products an instruction, each rounded.  (Sums of them stay single instructions: a
// packed sum would be fused with its products, and results would no longer be those of
// turn().)
__device__ __forceinline__ void mul2(float& r0, float& r1, float a0, float a1, float b0, float b1) {
    asm("{\n .reg .b64 a, b, r;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 r, a, b;\n"
        " mov.b64 {%0, %1}, r;\n}\n"
        : "=f"(r0), "=f"(r1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// Two pairs (a_i, b_i) turned.
__device__ __forceinline__ void turn2(float& a0, float& a1, float& b0, float& b1, float c0, float c1, float s0, float s1) {
    float ac0, ac1, bs0, bs1, bc0, bc1, as0, as1;
    mul2(ac0, ac1, a0, a1, c0, c1);
    mul2(bs0, bs1, b0, b1, s0, s1);
    mul2(bc0, bc1, b0, b1, c0, c1);
    mul2(as0, as1, a0, a1, s0, s1);
    a0 = __fsub_rn(ac0, bs0);
    a1 = __fsub_rn(ac1, bs1);
    b0 = __fadd_rn(bc0, as0);
    b1 = __fadd_rn(bc1, as1);
}

// The device's side of epq_pages.
struct PagesD {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    const int32_t* table;
    int64_t page_stride, scale_stride, table_stride, pages;
    int seqs, max_pages, page_size, kv_heads, head_dim, format;
    uint32_t page_mul, page_shift;

    // t / page_size for 0 <= t < 2^31 as a product (the constants: make_pages)
    __device__ __forceinline__ int page_of(int t) const {
        return (int)((__umulhi((uint32_t)t, page_mul) + (uint32_t)t) >> page_shift);
    }
};

// Page and slot of token `pos` of sequence `s`, or false with *bad set.
__device__ __forceinline__ bool find_slot(const PagesD& p, int s, int64_t pos, int64_t* page, int* slot, int* bad) {
    if (s < 0 || s >= p.seqs || pos >= (int64_t)p.max_pages * p.page_size) {
        *bad = kBadPosition;
        return false;
    }
    const int t = (int)pos;                       // max_pages * page_size < 2^31 (checked on the host)
    const int col = p.page_of(t);
    const int64_t pg = p.table[s * p.table_stride + col];
    if (pg < 0 || pg >= p.pages) {
        *bad = kBadPage;
        return false;
    }
    *page = pg;
    *slot = t - col * p.page_size;
    return true;
}

// Checks the description and copies it (k_paged_cache.cu).
int make_pages(const epq_pages* in, PagesD* out, const char* who);
// Whether rows of `v` can be read as `bytes`-byte words at every head and multiple of `bytes`.
inline bool heads_aligned(const epq_heads& v, int elem, int bytes) {
    return ((uintptr_t)v.data | (uintptr_t)(v.stride_row * elem) | (uintptr_t)(v.stride_head * elem)) % bytes == 0;
}

// Whether two heads of the view [m, heads, head_dim] have a value in common (an expanded tensor, say).
inline bool heads_overlap(const epq_heads& v, int64_t m, int64_t hd) {
    const int64_t H = v.heads;
    const int64_t sr = v.stride_row < 0 ? -v.stride_row : v.stride_row;
    const int64_t sh = v.stride_head < 0 ? -v.stride_head : v.stride_head;
    if ((m > 1 && sr < hd) || (H > 1 && sh < hd)) return true;
    if (m <= 1 || H <= 1 || sr / H >= sh || sh / m >= sr) return false;    // the ordinary orders: rows of heads, heads of rows
    for (int64_t h = 1; h < H; ++h) {
        const int64_t r = h * sh / sr, past = h * sh - r * sr;             // head h of row 0 begins `past` behind row r
        if ((r < m && past < hd) || (r + 1 < m && sr - past < hd)) return true;
    }
    return false;
}
// Whether y is written where x is read, but not value for value.
inline bool moved_in_place(const epq_heads& x, const epq_heads& y, int64_t m) {
    return x.data == y.data && ((m > 1 && x.stride_row != y.stride_row) || (x.heads > 1 && x.stride_head != y.stride_head));
}

int rope_read_device_error(int* flag);
int cache_read_device_error(int* flag);
int attend_read_device_error(int* flag);
int attend_blocks_read_device_error(int* flag);
int shared_read_device_error(int* flag);
int shared_read_timeout(int* flag);
int sparse_read_device_error(int* flag);

}  // namespace paged
}  // namespace epq
