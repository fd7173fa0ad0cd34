// kernels_norm.cu — the end of a residual block and the norm that opens the
// next, as one pass over the rows (lwm_gated_norm_device):
//   x' = x + rs * gate * post(y);  u = pre(x') (1 + scale) + shift;
//   h = LayerNorm(u) or u.
// Bound: memory; x and y are read once, x' and h written once.  A row lives
// in registers, 8 values a vector: 32 threads for widths up to 512 (one or two
// vectors a thread), 128 up to 1024, 256 above.  Means first, then squared
// differences, both in f32.
//
// Measured (one B200): 50176 rows of 1024, f32 stream and bf16 block, 617 MB
// in 116 us, 5.3 TB/s (a warp a row with four vectors a thread: 138); 1024
// rows of 192 in f32: 6.4 us, launch and one chain.  One barrier a sum
// instead of two, and streaming loads or stores, measured the same.
#include "lwm_blocks.cuh"

namespace lwm {

namespace {

__device__ __forceinline__ float load_one(const void* p, size_t at, int dtype) {
    if (dtype == LWM_DTYPE_F32) return static_cast<const float*>(p)[at];
    if (dtype == LWM_DTYPE_BF16) return __bfloat162float(static_cast<const bf16*>(p)[at]);
    return __half2float(static_cast<const __half*>(p)[at]);
}
__device__ __forceinline__ void store_one(void* p, size_t at, int dtype, float f) {
    if (dtype == LWM_DTYPE_F32) static_cast<float*>(p)[at] = f;
    else if (dtype == LWM_DTYPE_BF16) static_cast<bf16*>(p)[at] = __float2bfloat16_rn(f);
    else static_cast<__half*>(p)[at] = __float2half_rn(f);
}

// Sum over the row's threads; `red` holds a float per warp.
template <int kRow> __device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (kRow > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < kRow / 32; ++w) v += red[w];
    }
    return v;
}

// norm(v) * w + b over a row of `width` values, NV vectors of 8 a thread.
template <int kRow, int NV>
__device__ __forceinline__ void norm_row(float (&v)[NV][8], int kind, const float* w, const float* b, float eps,
                                         uint32_t width, uint32_t lane, float* red) {
    if (kind == LWM_NORM_NONE) return;
    const float inv_n = 1.0f / static_cast<float>(width);
    float mean = 0.0f;
    if (kind == LWM_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[q][e];  // vectors beyond the row are zero
        mean = row_sum<kRow>(s, red) * inv_n;
    }
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
        if ((lane + q * kRow) * 8 < width)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[q][e] -= mean;
                s += v[q][e] * v[q][e];
            }
    const float r = 1.0f / sqrtf(row_sum<kRow>(s, red) * inv_n + eps);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const uint32_t c = (lane + q * kRow) * 8;
        if (c >= width) continue;
        float t[8];
        if (w) {
            unpack(load8(w + c), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[q][e] *= r * t[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[q][e] *= r;
        }
        if (b) {
            unpack(load8(b + c), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[q][e] += t[e];
        }
    }
}

// Rows whose width is a multiple of 8 and whose buffers are 16-byte aligned;
// R, T, C: types of the residual stream, of y and h, and of the conditioning.
// Everything a row needs is asked for before any of it is used.
template <typename R, typename T, typename C, int kRow, int NV>
__global__ void __launch_bounds__(256) gated_norm_kernel(GatedNormArgs g) {
    __shared__ float red[8];
    const lwm_gated_norm_args& a = g.a;
    const uint32_t lane = threadIdx.x % kRow;
    const uint32_t r = blockIdx.x * (blockDim.x / kRow) + threadIdx.x / kRow;
    if (r >= a.rows) return;  // whole warps, or (kRow 256) never
    const size_t cond = static_cast<size_t>(g.cond_div.div(r)) * a.cond_stride;
    const R* xr = static_cast<const R*>(a.x) + r * a.x_stride;
    const T* yr = static_cast<const T*>(a.y) + r * a.y_stride;
    const C* gate = static_cast<const C*>(a.gate) + cond;
    Vec8<R> xv[NV];
    Vec8<T> yv[NV];
    Vec8<C> gv[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const uint32_t c = (lane + q * kRow) * 8;
        if (c >= a.width) continue;
        xv[q] = load8(xr + c);
        if (a.y) {
            yv[q] = load8(yr + c);
            if (a.gate) gv[q] = load8(gate + c);
        }
    }
    float x[NV][8];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[q][e] = 0.0f;
        if ((lane + q * kRow) * 8 < a.width) unpack(xv[q], x[q]);
    }
    if (a.y) {
        float y[NV][8];
#pragma unroll
        for (int q = 0; q < NV; ++q) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[q][e] = 0.0f;
            if ((lane + q * kRow) * 8 < a.width) unpack(yv[q], y[q]);
        }
        norm_row<kRow, NV>(y, a.post_kind, a.post_weight, a.post_bias, a.post_eps, a.width, lane, red);
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const uint32_t c = (lane + q * kRow) * 8;
            if (c >= a.width) continue;
            float t[8];
            if (a.residual_scale) {
                unpack(load8(a.residual_scale + c), t);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[q][e] *= t[e];
            }
            if (a.gate) {
                unpack(gv[q], t);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[q][e] *= t[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[q][e] += y[q][e];
        }
    }
    if (a.x_out) {
        R* out = static_cast<R*>(a.x_out) + r * a.x_out_stride;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const uint32_t c = (lane + q * kRow) * 8;
            if (c < a.width) store8(out + c, pack<R>(x[q]));
        }
    }
    if (!a.h) return;
    Vec8<C> sv[NV], bv[NV];
    const C *scale = static_cast<const C*>(a.scale) + cond, *shift = static_cast<const C*>(a.shift) + cond;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const uint32_t c = (lane + q * kRow) * 8;
        if (c < a.width && a.scale) sv[q] = load8(scale + c);
        if (c < a.width && a.shift) bv[q] = load8(shift + c);
    }
    norm_row<kRow, NV>(x, a.pre_kind, a.pre_weight, a.pre_bias, a.pre_eps, a.width, lane, red);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const uint32_t c = (lane + q * kRow) * 8;
        if (c >= a.width) continue;
        float t[8];
        if (a.scale) {
            unpack(sv[q], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[q][e] *= 1.0f + t[e];
        }
        if (a.shift) {
            unpack(bv[q], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[q][e] += t[e];
        }
    }
    if (g.out_norm)
        norm_row<kRow, NV>(x, LWM_NORM_LAYER, a.out_weight, a.out_bias, a.out_eps, a.width, lane, red);
    T* h = static_cast<T*>(a.h) + r * a.h_stride;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const uint32_t c = (lane + q * kRow) * 8;
        if (c < a.width) store8(h + c, pack<T>(x[q]));
    }
}

// Any width and alignment: a warp or a block a row, the row's values in shared
// memory.  us with the events around them: 20490 rows of 193, a warp each 51,
// a block each 103; of 1001, 139 and 190; but 100 rows of 1001, 35 and 23.
template <int kRow>
__device__ __forceinline__ void norm_smem(float* v, int kind, const float* w, const float* b, float eps, uint32_t width,
                                          uint32_t lane, float* red) {
    if (kind == LWM_NORM_NONE) return;
    const float inv_n = 1.0f / static_cast<float>(width);
    float mean = 0.0f;
    if (kind == LWM_NORM_LAYER) {
        float s = 0.0f;
        for (uint32_t i = lane; i < width; i += kRow) s += v[i];
        mean = row_sum<kRow>(s, red) * inv_n;
    }
    float s = 0.0f;
    for (uint32_t i = lane; i < width; i += kRow) {
        const float c = v[i] - mean;
        s += c * c;
    }
    const float r = 1.0f / sqrtf(row_sum<kRow>(s, red) * inv_n + eps);
    for (uint32_t i = lane; i < width; i += kRow) {
        float t = (v[i] - mean) * (w ? r * w[i] : r);
        if (b) t += b[i];
        v[i] = t;
    }
}
template <int kRow> __global__ void __launch_bounds__(256) gated_norm_any_kernel(GatedNormArgs g) {
    extern __shared__ float rows[];  // [rows of the block][width], each thread touches its own elements only
    __shared__ float red[8];
    const lwm_gated_norm_args& a = g.a;
    const uint32_t lane = threadIdx.x % kRow, r = blockIdx.x * (256 / kRow) + threadIdx.x / kRow;
    if (r >= a.rows) return;  // whole warps, or (kRow 256) never
    float* row = rows + threadIdx.x / kRow * a.width;
    const size_t cond = static_cast<size_t>(g.cond_div.div(r)) * a.cond_stride;
    if (a.y) {
        for (uint32_t i = lane; i < a.width; i += kRow) row[i] = load_one(a.y, r * a.y_stride + i, a.dtype);
        norm_smem<kRow>(row, a.post_kind, a.post_weight, a.post_bias, a.post_eps, a.width, lane, red);
    }
    for (uint32_t i = lane; i < a.width; i += kRow) {
        float x = load_one(a.x, r * a.x_stride + i, a.residual_dtype);
        if (a.y) {
            float y = row[i];
            if (a.residual_scale) y *= a.residual_scale[i];
            if (a.gate) y *= load_one(a.gate, cond + i, a.cond_dtype);
            x += y;
        }
        row[i] = x;
        if (a.x_out) store_one(a.x_out, r * a.x_out_stride + i, a.residual_dtype, x);
    }
    if (!a.h) return;
    norm_smem<kRow>(row, a.pre_kind, a.pre_weight, a.pre_bias, a.pre_eps, a.width, lane, red);
    for (uint32_t i = lane; i < a.width; i += kRow) {
        float u = row[i];
        if (a.scale) u *= 1.0f + load_one(a.scale, cond + i, a.cond_dtype);
        if (a.shift) u += load_one(a.shift, cond + i, a.cond_dtype);
        row[i] = u;
    }
    if (g.out_norm) norm_smem<kRow>(row, LWM_NORM_LAYER, a.out_weight, a.out_bias, a.out_eps, a.width, lane, red);
    for (uint32_t i = lane; i < a.width; i += kRow) store_one(a.h, r * a.h_stride + i, a.dtype, row[i]);
}

bool aligned(const void* p, uint64_t stride, size_t elem) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * elem % 16 == 0);
}

template <typename R, typename T, typename C, int kRow, int NV> cudaError_t launch_rows(const GatedNormArgs& g, cudaStream_t s) {
    const uint32_t per = kRow == 32 ? 4 : 1;  // rows a block
    gated_norm_kernel<R, T, C, kRow, NV><<<(g.a.rows + per - 1) / per, per * kRow, 0, s>>>(g);
    return cudaGetLastError();
}
template <typename R, typename T, typename C> cudaError_t launch_vectors(const GatedNormArgs& g, cudaStream_t s) {
    const uint32_t v = g.a.width / 8;
    if (v <= 32) return launch_rows<R, T, C, 32, 1>(g, s);
    if (v <= 64) return launch_rows<R, T, C, 32, 2>(g, s);
    if (v <= 128) return launch_rows<R, T, C, 128, 1>(g, s);
    if (v <= 256) return launch_rows<R, T, C, 256, 1>(g, s);
    if (v <= 512) return launch_rows<R, T, C, 256, 2>(g, s);
    return launch_rows<R, T, C, 256, 4>(g, s);
}

}  // namespace

cudaError_t launch_gated_norm(const GatedNormArgs& g, cudaStream_t s) {
    const lwm_gated_norm_args& a = g.a;
    const size_t re = a.residual_dtype == LWM_DTYPE_F32 ? 4 : 2, te = a.dtype == LWM_DTYPE_F32 ? 4 : 2,
                 ce = a.cond_dtype == LWM_DTYPE_F32 ? 4 : 2;
    const bool cond = a.gate || a.shift || a.scale;
    const bool vectors = a.width % 8 == 0 && aligned(a.x, a.x_stride, re) && aligned(a.x_out, a.x_out_stride, re) &&
                         aligned(a.y, a.y_stride, te) && aligned(a.h, a.h_stride, te) &&
                         aligned(a.gate, a.cond_stride, ce) && aligned(a.shift, a.cond_stride, ce) &&
                         aligned(a.scale, a.cond_stride, ce) && aligned(a.residual_scale, 0, 4) &&
                         aligned(a.post_weight, 0, 4) && aligned(a.post_bias, 0, 4) && aligned(a.pre_weight, 0, 4) &&
                         aligned(a.pre_bias, 0, 4) && aligned(a.out_weight, 0, 4) && aligned(a.out_bias, 0, 4);
    // the types that go together: a 32-bit residual stream or one in the block's type, conditioning likewise
    if (vectors) {
        const bool rf = a.residual_dtype == LWM_DTYPE_F32, cf = !cond || a.cond_dtype == LWM_DTYPE_F32;
        const bool rt = a.residual_dtype == a.dtype, ct = cond && a.cond_dtype == a.dtype;
        if (a.dtype == LWM_DTYPE_F32 && rf && cf) return launch_vectors<float, float, float>(g, s);
        if (a.dtype == LWM_DTYPE_BF16) {
            if (rf && cf) return launch_vectors<float, bf16, float>(g, s);
            if (rf && ct) return launch_vectors<float, bf16, bf16>(g, s);
            if (rt && cf) return launch_vectors<bf16, bf16, float>(g, s);
            if (rt && ct) return launch_vectors<bf16, bf16, bf16>(g, s);
        }
        if (a.dtype == LWM_DTYPE_F16) {
            if (rf && cf) return launch_vectors<float, __half, float>(g, s);
            if (rf && ct) return launch_vectors<float, __half, __half>(g, s);
            if (rt && cf) return launch_vectors<__half, __half, float>(g, s);
            if (rt && ct) return launch_vectors<__half, __half, __half>(g, s);
        }
    }
    if (a.width <= 256 || (a.width <= 1024 && a.rows >= 148 * 16))
        gated_norm_any_kernel<32><<<(a.rows + 7) / 8, 256, 8 * a.width * sizeof(float), s>>>(g);
    else
        gated_norm_any_kernel<256><<<a.rows, 256, a.width * sizeof(float), s>>>(g);
    return cudaGetLastError();
}

}  // namespace lwm
