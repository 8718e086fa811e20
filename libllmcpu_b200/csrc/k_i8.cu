// k_i8.cu -- a serving batch's rows in 8 bits: quantised with the norm before
// a projection, looked up from a table, and the entries of these and of the
// product (k_i8_linear.cu).
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdio>

#include "common.cuh"
#include "i8.h"
#include "i8_seen.h"

namespace nncu
{
namespace
{

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

constexpr int I8_COLS = 1 << 24; // the longest rows: their places stay far from 32 bits
constexpr float I8_TINY = 1.17549435e-38f; // 2^-126: the least step of a row's codes

// ---- quantise -------------------------------------------------------------------------
//
// Reads each value once and writes a byte; a value costs more than a dozen
// instructions, which memory does not hide, so that values go
// in pairs (one instruction for two), borders are settled for all of a thread's
// values at once, and the edges of a row are looked for once a thread. A row
// stays in the registers of `per_row` threads (16-byte loads) between its
// maximum and its codes; longer rows than a CTA holds are read twice. The
// squares of the norm are summed in 64 bits: float inputs' never overflow, and
// the scale is rounded once. 8191 x 2560 floats 18.8 us, with gain and norm 24.7
// (the copy rate: 16.0), bf16 17.6 and 22.3 (9.6): 23 instructions a value, issue
// slots 59 % busy. 16 values a thread and five CTAs of 256 threads per SM: with 32 values 51 us,
// with four CTAs 27, with CTAs that stay and copy ahead 29.

constexpr int Q_MOST = 256, Q_CTAS = 5; // threads of a row, and of a CTA; CTAs per SM
constexpr int Q_VALUES = 16; // a thread's values of a row (of a piece of it)

// VEC values at i, zeros past the row's end. FAST: rows on 16 bytes, a multiple of VEC long, so that all of them are there
// or none (code for odd ends beside it would be issued, without effect, for every value).
template <typename T, int VEC, bool FAST>
__device__ __forceinline__ void load_values(const T* x, int i, int cols, float* v)
{
	if constexpr (FAST)
	{
		uint4 q = make_uint4(0, 0, 0, 0);
		if (i < cols) q = *reinterpret_cast<const uint4*>(x + i);
		if constexpr (sizeof(T) == 4)
			v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
		else
		{
			const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
			for (int j = 0; j < 4; ++j)
			{
				const float2 f = widen2(w[j], static_cast<const T*>(nullptr));
				v[2 * j] = f.x, v[2 * j + 1] = f.y;
			}
		}
	}
	else
	{
#pragma unroll
		for (int j = 0; j < VEC; ++j) v[j] = i + j < cols ? load_elem(x + i + j) : 0.0f;
	}
}
// Their codes, out.
template <int VEC, bool FAST>
__device__ __forceinline__ void store_codes(int8_t* c, int i, int cols, const uint32_t* w)
{
	if constexpr (FAST)
	{
		if (i >= cols) return;
		if constexpr (VEC == 4)
			*reinterpret_cast<uint32_t*>(c + i) = w[0];
		else
			*reinterpret_cast<uint2*>(c + i) = make_uint2(w[0], w[1]);
	}
	else
#pragma unroll
		for (int j = 0; j < VEC; ++j)
			if (i + j < cols) c[i + j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
}

// The largest magnitude of a thread's values joins `most`, an infinity or a NaN makes `odd` a NaN (a maximum passes over NaN).
__device__ __forceinline__ void magnitudes(const float (&v)[Q_VALUES], float& most, float2& odd)
{
#pragma unroll
	for (int j = 0; j < Q_VALUES; j += 2)
	{
		most = fmaxf(most, fmaxf(fabsf(v[j]), fabsf(v[j + 1])));
		odd = fma2(make_float2(v[j], v[j + 1]), make_float2(0.0f, 0.0f), odd);
	}
}
// Its bits, which rise with it; above all numbers' where there was no number.
__device__ __forceinline__ uint32_t most_bits(float most, float2 odd)
{
	return odd.x + odd.y == 0.0f ? __float_as_uint(most) : 0x7F800000u;
}
__device__ __forceinline__ double squares(const float (&v)[Q_VALUES])
{
	double a = 0.0, b = 0.0;
#pragma unroll
	for (int j = 0; j < Q_VALUES; j += 2) a += (double)v[j] * v[j], b += (double)v[j + 1] * v[j + 1];
	return a + b;
}

__device__ __forceinline__ void times_gain(float* v, const float* g)
{
#pragma unroll
	for (int i = 0; i < 4; i += 2)
	{
		const float2 z = mul2(make_float2(v[i], v[i + 1]), make_float2(g[i], g[i + 1]));
		v[i] = z.x, v[i + 1] = z.y;
	}
}

constexpr float MAGIC = 12582912.0f; // 1.5 * 2^23: a sum's low bits are the rounded integer

// A thread's codes, x / s rounded to the nearest integer n, ties to even, four to a word. The quotient is corrected once, so
// that half integers come out as such and round to even. What is left of x, d = x - n s (exact: about s / 2 at most, in units
// of s's or x's last bit), then says whether n is right: where 2 |d| passes s (halving the least steps would round), x lies
// closer to a border than a float quotient tells, and n is one off. Of 32-bit inputs one in a million does: the largest |d|
// is returned, and i8_codes_exact writes such a thread's codes once more. Of 16-bit inputs one in two thousand does (their
// scale is a rounded one too): they are put right here.
template <bool NARROW>
__device__ __forceinline__ float i8_codes(const float (&v)[Q_VALUES], float s, float inv, bool bad, uint32_t (&w)[Q_VALUES / 4])
{
	uint32_t b[Q_VALUES];
	const float2 inv2 = make_float2(inv, inv), s2 = make_float2(-s, -s);
	float left = 0.0f;
#pragma unroll
	for (int j = 0; j < Q_VALUES; j += 2)
	{
		const float2 x = make_float2(v[j], v[j + 1]);
		float2 q = mul2(x, inv2);
		q = fma2(fma2(q, s2, x), inv2, q);
		const float2 t = add2(q, make_float2(MAGIC, MAGIC)), n = add2(t, make_float2(-MAGIC, -MAGIC)), d = fma2(n, s2, x);
		b[j] = __float_as_uint(t.x), b[j + 1] = __float_as_uint(t.y);
		left = fmaxf(left, fmaxf(fabsf(d.x), fabsf(d.y)));
	}
	if (NARROW)
	{
		if (__any_sync(0xffffffffu, left + left > s))
#pragma unroll
			for (int j = 0; j < Q_VALUES; ++j)
			{
				const float d = fmaf(-(__uint_as_float(b[j]) - MAGIC), s, v[j]);
				b[j] += (d + d > s) - (d + d < -s);
			}
	}
#pragma unroll
	for (int q = 0; q < Q_VALUES / 4; ++q) // (the low bytes)
		w[q] = bad ? 0u : __byte_perm(__byte_perm(b[4 * q], b[4 * q + 1], 0x0040), __byte_perm(b[4 * q + 2], b[4 * q + 3], 0x0040), 0x5410);
	return NARROW || bad ? 0.0f : left;
}

// A thread's codes of the piece of a row from p0 on, by what is left of each. (A call that reads its values anew, so that
// the common way holds nothing for it, and that takes them apart from the launch's struct, of which every thread would
// otherwise make a copy.)
template <typename T, bool FAST>
__device__ __noinline__ void i8_codes_exact(const T* x, const float* gamma, int8_t* codes, int cols, int p0, float s, float inv)
{
	constexpr int VEC = 16 / (int)sizeof(T), NV = Q_VALUES / VEC;
	float v[Q_VALUES];
	const auto place = [&](int k) { return p0 + (k * (int)blockDim.x + (int)threadIdx.x) * VEC; };
#pragma unroll
	for (int k = 0; k < NV; ++k) load_values<T, VEC, FAST>(x, place(k), cols, v + k * VEC);
	if (gamma)
#pragma unroll
		for (int j = 0; j < Q_VALUES; j += 4)
		{
			float g[4];
			load_values<float, 4, FAST>(gamma, place(j / VEC) + j % VEC, cols, g);
			times_gain(v + j, g);
		}
#pragma unroll
	for (int k = 0; k < NV; ++k)
	{
		uint32_t w[VEC / 4] = {};
#pragma unroll
		for (int j = 0; j < VEC; ++j)
		{
			const float z = v[k * VEC + j], t = z * inv + MAGIC, d = fmaf(-(t - MAGIC), s, z), d2 = d + d;
			uint32_t c = __float_as_uint(t);
			if (d2 > s || (d2 == s && (c & 1)))
				++c;
			else if (d2 < -s || (d2 == -s && (c & 1)))
				--c;
			w[j / 4] |= (c & 0xFFu) << (8 * (j % 4));
		}
		store_codes<VEC, FAST>(codes, place(k), cols, w);
	}
}

// The sum of n numbers in shared memory, on a warp.
__device__ __forceinline__ double sum_all(const double* p, int n)
{
	double s = 0.0;
	for (int i = (int)threadIdx.x % 32; i < n; i += 32) s += p[i];
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
	return s;
}

// The row's scale, rounded once; 1 / cols in 64 bits.
__device__ __forceinline__ float i8_scale(const nncu_i8_rows& r, double per_col, float s, bool bad, double sum)
{
	if (bad) return NAN;
	if (!r.norm) return s;
	const double mean = fma(sum, per_col, (double)r.eps);
	return mean > 0.0 ? (float)((double)s * rsqrt(mean)) : s;
}

// per_row threads of the CTA (x) take a row, blockDim.y rows a CTA; LOOP: rows longer than that.
template <typename T, bool FAST, bool LOOP>
__global__ void __launch_bounds__(Q_MOST, Q_CTAS) i8_quantise_kernel(const nncu_i8_rows r, double per_col)
{
	constexpr int V = Q_VALUES, VEC = 16 / (int)sizeof(T), NV = V / VEC;
	__shared__ uint32_t most_s[Q_MOST / 32];
	__shared__ double sum_s[Q_MOST];
	const int tid = (int)threadIdx.x, per_row = (int)blockDim.x, warps = per_row / 32;
	const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
	const bool live = row < r.n;
	const T* x = static_cast<const T*>(r.x) + (size_t)(live ? row : 0) * r.x_stride;
	const int piece = per_row * V, cols = live ? r.cols : 0;
	griddep_launch_dependents();
	griddep_wait();
	float v[V], most = 0.0f;
	float2 odd = make_float2(0.0f, 0.0f);
	double sum = 0.0;
	const auto load = [&](int p0) {
#pragma unroll
		for (int k = 0; k < NV; ++k) load_values<T, VEC, FAST>(x, p0 + (k * per_row + tid) * VEC, cols, v + k * VEC);
	};
	const auto gain = [&](int p0) {
		if (!r.gamma) return;
#pragma unroll
		for (int k = 0; k < NV; ++k)
#pragma unroll
			for (int j = 0; j < VEC; j += 4)
			{
				float g[4];
				load_values<float, 4, FAST>(r.gamma, p0 + (k * per_row + tid) * VEC + j, cols, g);
				times_gain(v + k * VEC + j, g);
			}
	};
	for (int p0 = 0; p0 < (LOOP ? cols : 1); p0 += piece)
	{
		load(p0);
		if (r.norm) sum += squares(v);
		gain(p0);
		magnitudes(v, most, odd);
	}
	uint32_t bits = __reduce_max_sync(0xffffffffu, most_bits(most, odd));
	const int at = (int)threadIdx.y * warps;
	if (r.norm) sum_s[(int)threadIdx.y * per_row + tid] = sum;
	if (warps > 1)
	{
		if (tid % 32 == 0) most_s[at + tid / 32] = bits;
		__syncthreads();
		bits = __reduce_max_sync(0xffffffffu, tid % 32 < warps ? most_s[at + tid % 32] : 0u);
	}
	else
		__syncwarp();
	const bool bad = bits >= 0x7F800000u;
	const float s = bad ? 1.0f : fmaxf(__fmul_rn(__uint_as_float(bits), 1.0f / 127.0f), I8_TINY), inv = __frcp_rn(s);
	int8_t* c = r.codes + (size_t)(live ? row : 0) * r.code_stride;
	for (int p0 = 0; p0 < (LOOP ? cols : 1); p0 += piece)
	{
		if (LOOP)
		{
			load(p0);
			gain(p0);
		}
		uint32_t w[V / 4];
		const float left = i8_codes<sizeof(T) == 2>(v, s, inv, bad, w);
#pragma unroll
		for (int k = 0; k < NV; ++k) store_codes<VEC, FAST>(c, p0 + (k * per_row + tid) * VEC, cols, w + k * (VEC / 4));
		if (sizeof(T) == 4 && live && left + left > s) i8_codes_exact<T, FAST>(x, r.gamma, c, cols, p0, s, inv);
	}
	if (tid < 32) // (one warp, after its codes: nobody waits for it)
	{
		if (r.norm) sum = sum_all(sum_s + (int)threadIdx.y * per_row, per_row);
		if (tid == 0 && live) r.scales[row] = i8_scale(r, per_col, s, bad, sum);
	}
}

// A launch that may begin while the one before it on the stream ends (its kernels wait for that end before they read).
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args)
{
	cudaLaunchAttribute at{};
	at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at.val.programmaticStreamSerializationAllowed = 1;
	cudaLaunchConfig_t cfg{};
	cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
	cfg.attrs = &at;
	cfg.numAttrs = 1;
	return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T>
int launch_quantise(const nncu_i8_rows& r, cudaStream_t st)
{
	const bool fast = (reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.gamma)) % 16 == 0 &&
	                  (r.n == 1 || r.x_stride * sizeof(T) % 16 == 0) && r.cols * sizeof(T) % 16 == 0;
	const int need = (r.cols + Q_VALUES - 1) / Q_VALUES, per_row = need > Q_MOST ? Q_MOST : (need + 31) / 32 * 32;
	const int rows = per_row >= 128 ? 1 : 128 / per_row; // short rows: several to a CTA
	const long long ctas = ((long long)r.n + rows - 1) / rows;
	const dim3 block(per_row, rows);
	if (need > Q_MOST)
		return launch_dependent(fast ? i8_quantise_kernel<T, true, true> : i8_quantise_kernel<T, false, true>, dim3((unsigned)ctas), block, 0, st, r, 1.0 / r.cols);
	return launch_dependent(fast ? i8_quantise_kernel<T, true, false> : i8_quantise_kernel<T, false, false>, dim3((unsigned)ctas), block, 0, st, r, 1.0 / r.cols);
}

// ---- look up ----------------------------------------------------------------------------
//
// Four bytes written for each one read: bound by the stores. A lane turns four
// codes into one 16-byte store, so that a warp's is 512 bytes in a row; four
// such loads are in flight a lane. A code becomes a float by putting it, as
// code + 128, below the bits of 2^23 and taking 2^23 + 128 off again. 8191 of
// 128256 x 2048: 15.0 us (the copy rate: 12.8); two loads a lane 16.8, eight 15.7.

constexpr int L_ITEMS = 4, L_MOST = 256;

// per_row threads of the CTA (x) take 16 values each of a row, blockDim.y rows a CTA; a row's next pieces along the grid's
// y. FAST: rows out on 16 bytes, a multiple of four long (as where rows are quantised).
template <bool FAST>
__global__ void __launch_bounds__(L_MOST) i8_lookup_kernel(const nncu_i8_lookup l)
{
	const long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
	griddep_launch_dependents();
	griddep_wait();
	if (t >= l.n) return;
	const int per_row = (int)blockDim.x, id = l.ids ? l.ids[t] : (int)t;
	const bool in = id >= 0 && id < l.n_rows;
	const int cols = l.cols, i0 = ((int)blockIdx.y * L_ITEMS * per_row + (int)threadIdx.x) * 4;
	const int8_t* c = l.codes + (size_t)(in ? id : 0) * l.code_stride + i0;
	float* out = l.out + (size_t)t * l.out_stride + i0;
	uint32_t w[L_ITEMS];
#pragma unroll
	for (int k = 0; k < L_ITEMS; ++k)
	{
		const int i = k * per_row * 4, left = in ? cols - i0 - i : 0;
		w[k] = 0;
		if (FAST)
		{
			if (left > 0) w[k] = *reinterpret_cast<const uint32_t*>(c + i);
		}
		else
#pragma unroll
			for (int j = 0; j < 4; ++j)
				if (j < left) w[k] |= (uint32_t)(uint8_t)c[i + j] << (8 * j);
	}
	const float s = in ? l.scales[id] * l.mult : 0.0f;
#pragma unroll
	for (int k = 0; k < L_ITEMS; ++k)
	{
		const int i = k * per_row * 4, left = cols - i0 - i;
		const uint32_t u = w[k] ^ 0x80808080u;
		const auto code = [&](int j) { return __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + j)); };
		const float2 off = make_float2(-8388736.0f, -8388736.0f), s2 = make_float2(s, s);
		const float2 a = mul2(add2(make_float2(code(0), code(1)), off), s2), b = mul2(add2(make_float2(code(2), code(3)), off), s2);
		if (FAST)
		{
			if (left > 0) *reinterpret_cast<float4*>(out + i) = make_float4(a.x, a.y, b.x, b.y);
		}
		else
		{
			const float v[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
			for (int j = 0; j < 4; ++j)
				if (j < left) out[i + j] = v[j];
		}
	}
}

int launch_lookup(const nncu_i8_lookup& l, cudaStream_t st)
{
	const bool fast = reinterpret_cast<uintptr_t>(l.out) % 16 == 0 && (l.n == 1 || l.out_stride % 4 == 0) && l.cols % 4 == 0;
	const int need = (l.cols + 4 * L_ITEMS - 1) / (4 * L_ITEMS), pieces = (need + L_MOST - 1) / L_MOST;
	const int per_row = ((need + pieces - 1) / pieces + 31) / 32 * 32; // the pieces alike: few idle threads
	const int rows = per_row >= 128 ? 1 : 128 / per_row;
	const dim3 grid((unsigned)(((long long)l.n + rows - 1) / rows), (unsigned)pieces), block(per_row, rows);
	return launch_dependent(fast ? i8_lookup_kernel<true> : i8_lookup_kernel<false>, grid, block, 0, st, l);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A stride that rows of `row` values fit, and whose product with a row's number stays far from 64 bits.
bool fits(size_t stride, int row) { return stride >= (size_t)row && stride <= (size_t)1 << 38; }

// `n` rows of `row` bytes, and the memory between the first byte and the last.
struct Span
{
	uintptr_t lo, hi;
	size_t n, stride, row;
};
Span span_bytes(const void* p, size_t n, size_t stride, size_t row)
{
	const uintptr_t a = reinterpret_cast<uintptr_t>(p);
	return {a, p && n ? a + (n - 1) * stride + row : a, n, stride, row};
}
// Whether two arrays have bytes in common. Rows equally far apart (or one row) may lie between the other's: columns of one
// buffer.
bool meet(const Span& a, const Span& b)
{
	if (a.hi <= b.lo || b.hi <= a.lo) return false;
	const size_t stride = a.n > 1 ? a.stride : b.stride;
	if ((a.n > 1 && b.n > 1 && a.stride != b.stride) || a.row > stride || b.row > stride) return true;
	const size_t d = b.lo >= a.lo ? (b.lo - a.lo) % stride : (stride - (a.lo - b.lo) % stride) % stride; // b's place behind a's
	return d < a.row || d + b.row > stride;
}

} // namespace

int check_current_device(std::initializer_list<const void*> arrays, const char* what)
{
	int dev = -1;
	cudaError_t ce = cudaGetDevice(&dev);
	for (const void* p : arrays)
	{
		if (!p) continue;
		cudaPointerAttributes at;
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
	}
	return NNCU_OK;
}

} // namespace nncu

using namespace nncu;

extern "C" int nncu_i8_quantise_dev(const nncu_i8_rows* r, void* stream)
{
	if (!r) return refuse("i8 quantise: NULL argument");
	if (r->n < 0 || r->cols <= 0 || r->cols > I8_COLS) return refuse("i8 quantise: bad n or cols (up to 2^24)");
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
	const int rc = check_current_device({r->x, r->gamma, r->codes, r->scales}, "i8 quantise");
	if (rc != NNCU_OK) return rc;
	const auto st = static_cast<cudaStream_t>(stream);
	const int e = r->x_type == NNCU_KV_F32    ? launch_quantise<float>(*r, st)
	              : r->x_type == NNCU_KV_BF16 ? launch_quantise<__nv_bfloat16>(*r, st)
	                                          : launch_quantise<__half>(*r, st);
	note_launches(1);
	if (e) cudaGetLastError();
	return e ? set_cuda_error(e, "i8 quantise launch") : NNCU_OK;
}

extern "C" int nncu_i8_lookup_dev(const nncu_i8_lookup* l, void* stream)
{
	if (!l) return refuse("i8 lookup: NULL argument");
	if (l->n < 0 || l->cols <= 0 || l->cols > I8_COLS || l->n_rows <= 0)
		return refuse("i8 lookup: bad n, cols (up to 2^24) or n_rows");
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
	const int rc = check_current_device({l->ids, l->codes, l->scales, l->out}, "i8 lookup");
	if (rc != NNCU_OK) return rc;
	const int e = launch_lookup(*l, static_cast<cudaStream_t>(stream));
	note_launches(1);
	if (e) cudaGetLastError();
	return e ? set_cuda_error(e, "i8 lookup launch") : NNCU_OK;
}

extern "C" int nncu_i8_linear_dev(const nncu_i8_linear* l, void* stream)
{
	if (!l) return refuse("i8 linear: NULL argument");
	if (l->n_tok < 0 || l->rows <= 0 || l->n_tok > 1 << 30 || l->rows > 1 << 30)
		return refuse("i8 linear: bad n_tok or rows (up to 2^30)");
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
	const int rc = check_current_device({l->x, l->x_scales, l->w, l->w_scales, l->bias, l->add, l->y}, "i8 linear");
	if (rc != NNCU_OK) return rc;
	const int e = launch_i8_linear(*l, stream);
	if (e) cudaGetLastError();
	note_launches(1);
	return e ? set_cuda_error(e, "i8 linear launch") : NNCU_OK;
}

extern "C" int nncu_i8_check(void* stream)
{
	static I8Seen seen;
	const auto st = static_cast<cudaStream_t>(stream);
	cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
	int dev = -1;
	unsigned long long id = 0;
	unsigned count = 0;
	cudaError_t ce = cudaStreamIsCapturing(st, &capturing);
	if (ce == cudaSuccess && capturing != cudaStreamCaptureStatusNone) return refuse("i8 check: the stream is being captured");
	if (ce == cudaSuccess) ce = cudaGetDevice(&dev);
	if (ce == cudaSuccess) ce = cudaStreamGetId(st, &id);
	// (a capture of another stream, which these calls do not concern, would be ended by them in its mode)
	cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
	if (ce == cudaSuccess) ce = cudaThreadExchangeStreamCaptureMode(&mode);
	if (ce == cudaSuccess)
	{
		ce = (cudaError_t)i8_waits_out(&count, stream);
		cudaThreadExchangeStreamCaptureMode(&mode);
	}
	if (ce != cudaSuccess)
	{
		cudaGetLastError();
		return set_cuda_error((int)ce, "i8 check");
	}
	return seen.more(dev, id, count)
	           ? set_error(NNCU_ERR_TIMEOUT, "an i8 product's bounded wait timed out; the outputs since this stream's last check are void")
	           : NNCU_OK;
}
