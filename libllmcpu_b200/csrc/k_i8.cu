// k_i8.cu -- a serving batch's rows in 8 bits: quantised with the norm before
// a projection, looked up from a table, and multiplied (nncu_i8_*).
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdio>

#include "common.cuh"
#include "i8.h"

namespace nncu
{
namespace
{

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

constexpr float I8_TINY = 1.17549435e-38f; // 2^-126: the least step of a row's codes

template <typename T>
__device__ __forceinline__ float block_reduce(float v, float* sm, T op)
{
	__syncthreads();
	sm[threadIdx.x] = v;
	__syncthreads();
	for (int o = blockDim.x / 2; o > 0; o >>= 1)
	{
		if ((int)threadIdx.x < o) sm[threadIdx.x] = op(sm[threadIdx.x], sm[threadIdx.x + o]);
		__syncthreads();
	}
	return sm[0];
}

// x / s rounded to the nearest integer, ties to even, exactly. The product with the reciprocal is at most one off next
// to a border; what is left of x then says which side it lies on (a fused multiply-add, exact here).
__device__ __forceinline__ float i8_code(float x, float s)
{
	float n = rintf(__fdiv_rn(x, s));
	const float d = fmaf(-n, s, x), h = 0.5f * s;
	if (d > h || (d == h && ((int)n & 1))) n += 1.0f;
	if (d < -h || (d == -h && ((int)n & 1))) n -= 1.0f;
	return n;
}

template <typename T>
__global__ void __launch_bounds__(256) i8_quantise_kernel(const nncu_i8_rows r)
{
	__shared__ float sm[256];
	__shared__ double sum;
	const size_t t = blockIdx.x;
	const T* x = static_cast<const T*>(r.x) + t * r.x_stride;
	float most = 0.0f;
	double ss = 0.0;
	bool bad = false;
	for (int i = threadIdx.x; i < r.cols; i += 256)
	{
		const float v = load_elem(x + i), z = r.gamma ? v * r.gamma[i] : v;
		most = fmaxf(most, fabsf(z));
		bad |= !(fabsf(z) < INFINITY);
		ss += (double)v * v;
	}
	if (threadIdx.x == 0) sum = 0.0;
	bad = __syncthreads_or(bad);
	atomicAdd(&sum, ss);
	most = block_reduce(most, sm, [](float a, float b) { return fmaxf(a, b); });
	const float s = fmaxf(__fdiv_rn(most, 127.0f), I8_TINY);
	const double mean = sum / r.cols + (double)r.eps;
	if (threadIdx.x == 0)
		r.scales[t] = bad ? NAN : r.norm && mean > 0.0 ? (float)((double)s / sqrt(mean)) : s;
	int8_t* c = r.codes + t * r.code_stride;
	for (int i = threadIdx.x; i < r.cols; i += 256)
	{
		const float v = load_elem(x + i), z = r.gamma ? v * r.gamma[i] : v;
		c[i] = bad ? 0 : (int8_t)(int)i8_code(z, s);
	}
}

__global__ void __launch_bounds__(256) i8_lookup_kernel(const nncu_i8_lookup l)
{
	const size_t t = blockIdx.x;
	const int id = l.ids ? l.ids[t] : (int)t;
	const bool in = id >= 0 && id < l.n_rows;
	const float s = in ? l.scales[id] * l.mult : 0.0f;
	const int8_t* c = l.codes + (size_t)(in ? id : 0) * l.code_stride;
	for (int i = threadIdx.x; i < l.cols; i += 256) l.out[t * l.out_stride + i] = in ? s * (float)c[i] : 0.0f;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A stride that rows of `row` values fit, and whose product with a row's number stays far from 64 bits.
bool fits(size_t stride, int row) { return stride >= (size_t)row && stride <= (size_t)1 << 38; }

// The memory between the first byte of `n` rows and the last.
struct Span
{
	uintptr_t lo, hi;
};
Span span_bytes(const void* p, size_t n, size_t stride, size_t row)
{
	const uintptr_t a = reinterpret_cast<uintptr_t>(p);
	return {a, p && n ? a + (n - 1) * stride + row : a};
}
bool meet(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

} // namespace

int check_current_device(const void* p, const char* what)
{
	int dev = -1;
	cudaPointerAttributes at;
	cudaError_t ce = cudaGetDevice(&dev);
	if (ce == cudaSuccess) ce = cudaPointerGetAttributes(&at, p);
	if (ce != cudaSuccess)
	{
		cudaGetLastError();
		return set_cuda_error((int)ce, what);
	}
	if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
	{
		char msg[120];
		snprintf(msg, sizeof msg, "%s: the arrays must be device memory", what);
		return refuse(msg);
	}
	if (at.device != dev)
	{
		char msg[120];
		snprintf(msg, sizeof msg, "%s: the arrays lie on device %d, the current one is %d", what, at.device, dev);
		return refuse(msg);
	}
	return NNCU_OK;
}

} // namespace nncu

using namespace nncu;

extern "C" int nncu_i8_quantise_dev(const nncu_i8_rows* r, void* stream)
{
	if (!r) return refuse("i8 quantise: NULL argument");
	if (r->n < 0 || r->cols <= 0) return refuse("i8 quantise: bad n or cols");
	if (r->x_type != NNCU_KV_F32 && r->x_type != NNCU_KV_BF16 && r->x_type != NNCU_KV_F16)
		return refuse("i8 quantise: unknown x_type");
	if (r->norm && !(r->eps >= 0.0f && r->eps < INFINITY)) return refuse("i8 quantise: eps must be finite and not negative");
	if (r->n == 0) return NNCU_OK;
	if (!r->x || !r->codes || !r->scales) return refuse("i8 quantise: NULL array");
	const size_t esize = r->x_type == NNCU_KV_F32 ? 4 : 2;
	if (reinterpret_cast<uintptr_t>(r->x) % esize || reinterpret_cast<uintptr_t>(r->scales) % 4 ||
	    reinterpret_cast<uintptr_t>(r->gamma) % 4)
		return refuse("i8 quantise: x, gamma or scales not aligned to their type");
	if (!aligned16(r->codes) || (r->n > 1 && r->code_stride % 16))
		return refuse("i8 quantise: rows of codes must be 16-byte aligned");
	if (r->n > 1 && (!fits(r->x_stride, r->cols) || !fits(r->code_stride, r->cols)))
		return refuse("i8 quantise: strides shorter than a row or past 2^38");
	const Span x = span_bytes(r->x, r->n, r->x_stride * esize, r->cols * esize), g = span_bytes(r->gamma, 1, 0, 4 * (size_t)r->cols),
	           c = span_bytes(r->codes, r->n, r->code_stride, r->cols), s = span_bytes(r->scales, r->n, 4, 4);
	if (meet(c, x) || meet(s, x) || meet(c, s) || meet(c, g) || meet(s, g))
		return refuse("i8 quantise: codes and scales must not meet another array");
	const int rc = check_current_device(r->codes, "i8 quantise");
	if (rc != NNCU_OK) return rc;
	const auto st = static_cast<cudaStream_t>(stream);
	if (r->x_type == NNCU_KV_F32)
		i8_quantise_kernel<float><<<r->n, 256, 0, st>>>(*r);
	else if (r->x_type == NNCU_KV_BF16)
		i8_quantise_kernel<__nv_bfloat16><<<r->n, 256, 0, st>>>(*r);
	else
		i8_quantise_kernel<__half><<<r->n, 256, 0, st>>>(*r);
	note_launches(1);
	const int e = (int)cudaGetLastError();
	return e ? set_cuda_error(e, "i8 quantise launch") : NNCU_OK;
}

extern "C" int nncu_i8_lookup_dev(const nncu_i8_lookup* l, void* stream)
{
	if (!l) return refuse("i8 lookup: NULL argument");
	if (l->n < 0 || l->cols <= 0 || l->n_rows <= 0) return refuse("i8 lookup: bad n, cols or n_rows");
	if (!l->ids && l->n > l->n_rows) return refuse("i8 lookup: more rows than the table has, without ids");
	if (!std::isfinite(l->mult)) return refuse("i8 lookup: mult must be finite");
	if (l->n == 0) return NNCU_OK;
	if (!l->codes || !l->scales || !l->out) return refuse("i8 lookup: NULL array");
	if (reinterpret_cast<uintptr_t>(l->ids) % 4 || reinterpret_cast<uintptr_t>(l->scales) % 4 ||
	    reinterpret_cast<uintptr_t>(l->out) % 4)
		return refuse("i8 lookup: ids, scales or out not aligned to their type");
	if (!aligned16(l->codes) || (l->n_rows > 1 && l->code_stride % 16))
		return refuse("i8 lookup: rows of codes must be 16-byte aligned");
	if ((l->n_rows > 1 && !fits(l->code_stride, l->cols)) || (l->n > 1 && !fits(l->out_stride, l->cols)))
		return refuse("i8 lookup: strides shorter than a row or past 2^38");
	const Span o = span_bytes(l->out, l->n, l->out_stride * 4, 4 * (size_t)l->cols);
	if (meet(o, span_bytes(l->codes, l->n_rows, l->code_stride, l->cols)) || meet(o, span_bytes(l->scales, l->n_rows, 4, 4)) ||
	    meet(o, span_bytes(l->ids, l->n, 4, 4)))
		return refuse("i8 lookup: out must not meet another array");
	const int rc = check_current_device(l->out, "i8 lookup");
	if (rc != NNCU_OK) return rc;
	i8_lookup_kernel<<<l->n, 256, 0, static_cast<cudaStream_t>(stream)>>>(*l);
	note_launches(1);
	const int e = (int)cudaGetLastError();
	return e ? set_cuda_error(e, "i8 lookup launch") : NNCU_OK;
}

extern "C" int nncu_i8_linear_dev(const nncu_i8_linear* l, void* stream)
{
	if (!l) return refuse("i8 linear: NULL argument");
	if (l->n_tok < 0 || l->rows <= 0) return refuse("i8 linear: bad n_tok or rows");
	if (l->cols <= 0 || l->cols > 131071) return refuse("i8 linear: cols must be 1 to 131071"); // (2^14 cols < 2^31)
	if ((long long)l->n_tok * l->rows > (1ll << 36)) return refuse("i8 linear: n_tok * rows passes 2^36");
	if (l->n_tok == 0) return NNCU_OK;
	if (!l->x || !l->x_scales || !l->w || !l->w_scales || !l->y) return refuse("i8 linear: NULL array");
	if (!aligned16(l->x) || !aligned16(l->w) || (l->n_tok > 1 && l->x_stride % 16) || (l->rows > 1 && l->w_stride % 16))
		return refuse("i8 linear: rows of codes must be 16-byte aligned");
	if ((reinterpret_cast<uintptr_t>(l->x_scales) | reinterpret_cast<uintptr_t>(l->w_scales) | reinterpret_cast<uintptr_t>(l->bias) |
	     reinterpret_cast<uintptr_t>(l->add) | reinterpret_cast<uintptr_t>(l->y)) % 4)
		return refuse("i8 linear: scales, bias, add or y not aligned to their type");
	if ((l->n_tok > 1 && (!fits(l->x_stride, l->cols) || !fits(l->y_stride, l->rows) || (l->add && !fits(l->add_stride, l->rows)))) ||
	    (l->rows > 1 && !fits(l->w_stride, l->cols)))
		return refuse("i8 linear: strides shorter than a row or past 2^38");
	const size_t row = 4 * (size_t)l->rows;
	const Span y = span_bytes(l->y, l->n_tok, l->y_stride * 4, row);
	const bool in_place = l->add == l->y && (l->n_tok == 1 || l->add_stride == l->y_stride);
	if (meet(y, span_bytes(l->x, l->n_tok, l->x_stride, l->cols)) || meet(y, span_bytes(l->w, l->rows, l->w_stride, l->cols)) ||
	    meet(y, span_bytes(l->x_scales, l->n_tok, 4, 4)) || meet(y, span_bytes(l->w_scales, l->rows, 4, 4)) ||
	    meet(y, span_bytes(l->bias, 1, 0, row)) || (!in_place && meet(y, span_bytes(l->add, l->n_tok, l->add_stride * 4, row))))
		return refuse("i8 linear: y must not meet an input (add may be y itself)");
	const int rc = check_current_device(l->y, "i8 linear");
	if (rc != NNCU_OK) return rc;
	const int e = launch_i8_linear(*l, stream);
	if (e) cudaGetLastError();
	note_launches(1);
	return e ? set_cuda_error(e, "i8 linear launch") : NNCU_OK;
}

extern "C" int nncu_i8_check(void* stream)
{
	int word = 0;
	cudaError_t ce = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
	if (ce == cudaSuccess) ce = (cudaError_t)i8_error_word(&word);
	if (ce != cudaSuccess) return set_cuda_error((int)ce, "i8 check");
	return word ? set_error(NNCU_ERR_TIMEOUT, "an i8 product's bounded wait timed out; the outputs since the last check are void") : NNCU_OK;
}
