// k_logprobs.cu -- what a server reports of rows of logits (nncu_logprobs_dev):
// log probabilities of given tokens, their ranks, entropies, the likeliest
// tokens.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cfloat>

#include "common.cuh"
#include "nncu.h"

namespace nncu
{
namespace
{

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

constexpr int LP_THREADS = 256, LP_TOP = 32;

// Keys that order logits downwards and equal ones by their index: the larger key comes first. A NaN counts as
// -infinity, both zeros alike. The lowest key of all is 0 (no logit has it).
__device__ __forceinline__ unsigned long long lp_key(float x, int i)
{
	const uint32_t b = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
	const uint32_t u = b & 0x80000000u ? ~b : b | 0x80000000u;
	return (unsigned long long)u << 32 | (0xFFFFFFFFu - (uint32_t)i);
}

__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const nncu_logprobs l)
{
	__shared__ double sm[LP_THREADS], sh[LP_THREADS];
	__shared__ float mx[LP_THREADS];
	__shared__ int before;
	__shared__ unsigned long long best[LP_THREADS];
	const size_t r = blockIdx.x;
	const float* x = l.logits + r * l.stride;
	const int tok = l.tokens ? l.tokens[r] : -1, n = l.n_vocab;
	const bool in = tok >= 0 && tok < n;
	if (threadIdx.x == 0) before = 0;
	float m = -FLT_MAX;
	for (int i = threadIdx.x; i < n; i += LP_THREADS) m = fmaxf(m, x[i]);
	mx[threadIdx.x] = m;
	__syncthreads();
	for (int o = LP_THREADS / 2; o > 0; o >>= 1)
	{
		if ((int)threadIdx.x < o) mx[threadIdx.x] = fmaxf(mx[threadIdx.x], mx[threadIdx.x + o]);
		__syncthreads();
	}
	m = mx[0];
	double z = 0.0, h = 0.0;
	int rank = 0;
	const unsigned long long mine = in ? lp_key(x[tok], tok) : 0;
	for (int i = threadIdx.x; i < n; i += LP_THREADS)
	{
		const float t = (x[i] - m) * l.scale, e = expf(t);
		z += e;
		h += e > 0.0f ? e * t : 0.0f;
		rank += lp_key(x[i], i) > mine;
	}
	sm[threadIdx.x] = z, sh[threadIdx.x] = h;
	atomicAdd(&before, rank);
	__syncthreads();
	for (int o = LP_THREADS / 2; o > 0; o >>= 1)
	{
		if ((int)threadIdx.x < o) sm[threadIdx.x] += sm[threadIdx.x + o], sh[threadIdx.x] += sh[threadIdx.x + o];
		__syncthreads();
	}
	z = sm[0], h = sh[0];
	const double lz = log(z);
	if (threadIdx.x == 0)
	{
		if (l.logprob) l.logprob[r] = in ? (z == 0.0 ? -INFINITY : (float)((double)((x[tok] - m) * l.scale) - lz)) : 0.0f;
		if (l.rank) l.rank[r] = in ? before : -1;
		if (l.entropy) l.entropy[r] = z == 0.0 ? 0.0f : (float)(lz - h / z);
	}
	unsigned long long below = ~0ull;
	for (int k = 0; k < l.top; ++k)
	{
		unsigned long long b = 0;
		for (int i = threadIdx.x; i < n; i += LP_THREADS)
		{
			const unsigned long long q = lp_key(x[i], i);
			if (q < below && q > b) b = q;
		}
		__syncthreads();
		best[threadIdx.x] = b;
		__syncthreads();
		for (int o = LP_THREADS / 2; o > 0; o >>= 1)
		{
			if ((int)threadIdx.x < o && best[threadIdx.x + o] > best[threadIdx.x]) best[threadIdx.x] = best[threadIdx.x + o];
			__syncthreads();
		}
		below = best[0];
		if (threadIdx.x == 0)
		{
			const int id = (int)(0xFFFFFFFFu - (uint32_t)below);
			const bool live = (below >> 32) > 0x007FFFFFu; // above -infinity
			if (l.top_ids) l.top_ids[r * l.top + k] = live ? id : -1;
			if (l.top_logprobs) l.top_logprobs[r * l.top + k] = live ? (float)((double)((x[id] - m) * l.scale) - lz) : -INFINITY;
		}
	}
}

} // namespace
} // namespace nncu

using namespace nncu;

extern "C" int nncu_logprobs_dev(const nncu_logprobs* l, void* stream)
{
	if (!l) return refuse("logprobs: NULL argument");
	if (l->n < 0 || l->n_vocab <= 0) return refuse("logprobs: bad n or n_vocab");
	if (l->top < 0 || l->top > LP_TOP || l->top > l->n_vocab) return refuse("logprobs: top must be 0 to 32, n_vocab at most");
	if (!(l->scale > 0.0f && l->scale < INFINITY)) return refuse("logprobs: scale must be finite and above zero");
	if (l->n == 0) return NNCU_OK;
	if (!l->logits) return refuse("logprobs: NULL logits");
	if ((l->logprob || l->rank) && !l->tokens) return refuse("logprobs: logprob and rank need tokens");
	if (!l->logprob && !l->rank && !l->entropy && !(l->top && (l->top_ids || l->top_logprobs)))
		return refuse("logprobs: no output");
	if (l->n > 1 && (l->stride < (size_t)l->n_vocab || l->stride > (size_t)1 << 38))
		return refuse("logprobs: stride shorter than a row or past 2^38");
	const void* all[] = {l->logits, l->tokens, l->logprob, l->rank, l->entropy, l->top_ids, l->top_logprobs};
	for (const void* p : all)
		if (reinterpret_cast<uintptr_t>(p) % 4) return refuse("logprobs: an array is not aligned to its type");
	// outputs that meet one another or an input
	struct
	{
		uintptr_t lo, hi;
	} s[7];
	const size_t len[] = {(size_t)(l->n - 1) * l->stride + l->n_vocab, (size_t)l->n, (size_t)l->n, (size_t)l->n, (size_t)l->n,
	                      (size_t)l->n * l->top, (size_t)l->n * l->top};
	for (int i = 0; i < 7; ++i)
	{
		s[i].lo = reinterpret_cast<uintptr_t>(all[i]);
		s[i].hi = all[i] ? s[i].lo + 4 * len[i] : s[i].lo;
		for (int j = 0; j < i; ++j)
			if (i > 1 && s[i].lo < s[j].hi && s[j].lo < s[i].hi) return refuse("logprobs: outputs must not meet another array");
	}
	const int rc = check_current_device(l->logits, "logprobs");
	if (rc != NNCU_OK) return rc;
	logprobs_kernel<<<l->n, LP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*l);
	note_launches(1);
	const int e = (int)cudaGetLastError();
	return e ? set_cuda_error(e, "logprobs launch") : NNCU_OK;
}
