// k_logprobs.cu -- what a server reports of rows of logits (nncu_logprobs_dev):
// log probabilities of given tokens, their ranks, entropies, the likeliest
// tokens.
//
// Mathematics. One pass over a row, in base 2 with k = scale / ln 2: a thread
// holds the largest logit m that it has met, z = sum 2^((x - m) k) and h = sum
// 2^((x - m) k) (x - m) k, moved to a new m when one comes; parts join the same
// way. Then log p(x) = (x - m) scale - ln z and the entropy is ln z - h ln 2 / z.
// The rank counts logits above the token's while they pass.
//
// The likeliest tokens need no second pass: a thread remembers its largest
// logit and the largest outside of that one's group. The top-th of the threads'
// largest bounds the answer from below, so that `top` threads at most can hold
// any of it, and nearly always one each: their groups are read again (16
// logits), the rest of a thread's share only where its second group passes the bound.
//
// Bound by memory where rows are many; a row is shared by up to eight CTAs (a
// cluster, whose parts meet in shared memory) where they are few.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "nncu.h"

namespace nncu
{
namespace
{

__device__ __forceinline__ void cluster_sync()
{
	asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The generic address of `p` (this CTA's shared memory) in the cluster's CTA `rank`.
__device__ __forceinline__ const void* cluster_map(const void* p, int rank)
{
	uint64_t r;
	asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
	return reinterpret_cast<const void*>(r);
}

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32, LP_TOP = 32;
constexpr int LP_ITEMS = 4;                      // 16-byte loads a thread has in flight
constexpr int LP_GROUP = LP_THREADS * LP_ITEMS;  // vectors (of four logits) that the CTA takes at a time
constexpr int LP_CLUSTER = 8;                    // the most CTAs that share a row
constexpr int LP_FOUND = LP_TOP * 4 * LP_ITEMS + LP_WARPS * LP_TOP;

using Key = unsigned long long;

// Keys that order logits downwards and equal ones by their index: the larger key comes first. Both zeros are alike. 0 is
// below all of them, and stands for a logit that is no candidate: masked, or a NaN.
__device__ __forceinline__ Key lp_key(float x, int i)
{
	if (!(x > -INFINITY)) return 0;
	const uint32_t b = __float_as_uint(x + 0.0f);
	const uint32_t u = b & 0x80000000u ? ~b : b | 0x80000000u;
	return (Key)u << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float lp_value(Key k)
{
	const uint32_t u = (uint32_t)(k >> 32);
	return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int lp_index(Key k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

// One step of a bitonic sort over the warp: each lane keeps the larger or the smaller of its key and its partner's.
__device__ __forceinline__ Key lp_step(Key k, int mask, bool larger)
{
	const Key o = __shfl_xor_sync(0xffffffffu, k, mask);
	return (k > o) == larger ? k : o;
}
// The warp's keys in falling order.
__device__ __forceinline__ Key lp_sort(Key k, int lane)
{
#pragma unroll
	for (int size = 2; size <= 32; size *= 2)
#pragma unroll
		for (int d = size / 2; d > 0; d /= 2) k = lp_step(k, d, ((lane & d) == 0) == ((lane & size) == 0));
	return k;
}
// The 32 largest of two falling runs of 32, falling.
__device__ __forceinline__ Key lp_merge(Key a, Key b, int lane)
{
	const Key r = __shfl_sync(0xffffffffu, b, 31 - lane);
	a = a > r ? a : r;
#pragma unroll
	for (int d = 16; d > 0; d /= 2) a = lp_step(a, d, (lane & d) == 0);
	return a;
}

// What a part of a row knows of its softmax, in base 2: the largest logit, the sum of e = 2^((x - m) k) and that of e
// times its exponent.
struct Stat
{
	float m, z, h;
};
__device__ __forceinline__ Stat lp_join(Stat a, Stat b, float k)
{
	const float m = fmaxf(a.m, b.m);
	// (held above -infinity, so that an empty part adds zeros)
	const float da = fmaxf((a.m - m) * k, -1e5f), db = fmaxf((b.m - m) * k, -1e5f);
	const float ca = ex2(da), cb = ex2(db);
	return {m, a.z * ca + b.z * cb, ca * (a.h + da * a.z) + cb * (b.h + db * b.z)};
}
__device__ __forceinline__ Stat lp_shfl(Stat s, int d)
{
	return {__shfl_xor_sync(0xffffffffu, s.m, d), __shfl_xor_sync(0xffffffffu, s.z, d), __shfl_xor_sync(0xffffffffu, s.h, d)};
}

struct LpArgs
{
	nncu_logprobs l;
	float k; // scale / ln 2
	int parts;
};

// What a CTA hands to the one that finishes its row.
struct Part
{
	Key top[LP_TOP];
	Stat stat;
	int before;
};

template <bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 2) logprobs_kernel(const LpArgs a)
{
	__shared__ Part mine;
	__shared__ Stat warp_stat[LP_WARPS];
	__shared__ int warp_before[LP_WARPS];
	__shared__ Key lists[TOP ? LP_WARPS : 1][LP_TOP], found[TOP ? LP_FOUND : 1];
	__shared__ int n_found, n_again;
	__shared__ short again[TOP ? LP_TOP : 1];
	const nncu_logprobs& l = a.l;
	const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int part = (int)(blockIdx.x % a.parts);
	const size_t r = blockIdx.x / a.parts;
	const int n = l.n_vocab;
	const float* x = l.logits + r * l.stride;
	// Vectors of four logits lie on 16 bytes: the row's first and last one may be cut.
	const int cut = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
	const float* base = x - cut;
	const int nvec = (n + cut + 3) / 4, each = (nvec + a.parts - 1) / a.parts;
	const int v0 = min(nvec, part * each), v1 = min(nvec, v0 + each);
	const float k = a.k;

	const int tok = l.tokens ? l.tokens[r] : -1;
	const bool in = tok >= 0 && tok < n;
	const float xt = in ? x[tok] : 0.0f;
	const bool hidden = in && !(xt > -INFINITY);      // (a NaN comes as -infinity)
	const float below = nextafterf(xt, -INFINITY);    // x >= xt is x > below
	const int tok_vec = in ? (tok + cut) / 4 : -1;

	const auto load = [&](int j) {
		if (j > 0 && j < nvec - 1) return __ldg(reinterpret_cast<const float4*>(base) + j);
		float v[4];
#pragma unroll
		for (int c = 0; c < 4; ++c)
		{
			const int i = 4 * j + c - cut;
			v[c] = i >= 0 && i < n ? __ldg(x + i) : -INFINITY;
		}
		return make_float4(v[0], v[1], v[2], v[3]);
	};

	Stat s{-FLT_MAX, 0.0f, 0.0f};
	int before = 0;
	float best = -INFINITY, second = -INFINITY; // the largest of the thread's groups, and of the others
	int best_at = v0;
	for (int g = v0; g < v1; g += LP_GROUP)
	{
		float4 q[LP_ITEMS];
		if (g > 0 && g + LP_GROUP <= v1 && g + LP_GROUP < nvec)
		{
#pragma unroll
			for (int u = 0; u < LP_ITEMS; ++u) q[u] = __ldg(reinterpret_cast<const float4*>(base) + g + u * LP_THREADS + tid);
		}
		else
		{
#pragma unroll
			for (int u = 0; u < LP_ITEMS; ++u)
			{
				const int j = g + u * LP_THREADS + tid;
				q[u] = j < v1 ? load(j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
			}
		}
		float top = -INFINITY;
#pragma unroll
		for (int u = 0; u < LP_ITEMS; ++u) top = fmaxf(top, fmaxf(fmaxf(q[u].x, q[u].y), fmaxf(q[u].z, q[u].w)));
		if (TOP)
		{
			if (top > best)
				second = best, best = top, best_at = g;
			else
				second = fmaxf(second, top);
		}
		if (top > s.m)
		{
			const float d = fmaxf((s.m - top) * k, -1e5f), c = ex2(d);
			s.h = c * (s.h + d * s.z);
			s.z *= c;
			s.m = top;
		}
		float z = 0.0f, h = 0.0f;
#pragma unroll
		for (int u = 0; u < LP_ITEMS; ++u)
		{
			const float v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
			const int j = g + u * LP_THREADS + tid;
			const float over = j < tok_vec ? below : xt;
#pragma unroll
			for (int c = 0; c < 4; ++c)
			{
				const float t = (v[c] - s.m) * k, e = ex2(t);
				z += e;
				h = fmaf(e, fmaxf(t, -200.0f), h); // (2^-200 is 0: what is masked adds no 0 * infinity)
				before += v[c] > over;
			}
		}
		s.z += z;
		s.h += h;
		if (hidden) // every token that is not masked comes before a masked one, and the masked ones before it
		{
#pragma unroll
			for (int u = 0; u < LP_ITEMS; ++u)
			{
				const float v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
				const int j = g + u * LP_THREADS + tid;
#pragma unroll
				for (int c = 0; c < 4; ++c)
				{
					const int i = 4 * j + c - cut;
					before -= v[c] > (j < tok_vec ? below : xt);
					before += j < v1 && i >= 0 && i < n && (v[c] > -INFINITY || i < tok);
				}
			}
		}
	}
	// equal ones before the token in its own vector
	if (in && !hidden && tid == 0 && tok_vec >= v0 && tok_vec < v1)
		for (int i = max(0, 4 * tok_vec - cut); i < tok; ++i) before += x[i] == xt;

#pragma unroll
	for (int d = 16; d > 0; d >>= 1) s = lp_join(s, lp_shfl(s, d), k);
	before = __reduce_add_sync(0xffffffffu, before);
	if (lane == 0) warp_stat[warp] = s, warp_before[warp] = before;
	if (tid == 0) n_found = n_again = 0;

	if (TOP)
	{
		// The thread's first candidate: the first of its largest logits, in the group that reached them first.
		float4 q[LP_ITEMS];
#pragma unroll
		for (int u = 0; u < LP_ITEMS; ++u)
		{
			const int j = best_at + u * LP_THREADS + tid;
			q[u] = best > -INFINITY && j < v1 ? load(j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
		}
		Key first = 0;
#pragma unroll
		for (int u = LP_ITEMS - 1; u >= 0; --u)
		{
			const float v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
			for (int c = 3; c >= 0; --c)
				if (v[c] == best) first = lp_key(best, 4 * (best_at + u * LP_THREADS + tid) + c - cut);
		}
		// The CTA's top tokens are not before the top-th of the threads' firsts, and lie with the threads whose own
		// first is not after that one: `top` threads at most.
		Key list = lp_sort(first, lane);
		lists[warp][lane] = list;
		__syncthreads();
#pragma unroll
		for (int d = LP_WARPS / 2; d > 0; d /= 2)
		{
			if (warp < d) lists[warp][lane] = list = lp_merge(list, lists[warp + d][lane], lane);
			__syncthreads();
		}
		const Key least = lists[0][l.top - 1];
		if (first != 0 && first >= least)
		{
			if (least == 0 ? second > -INFINITY : second >= lp_value(least)) // more of them may lie in the thread's other groups
				again[atomicAdd(&n_again, 1)] = (short)tid;
			else
#pragma unroll
				for (int u = 0; u < LP_ITEMS; ++u)
				{
					const float v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
					for (int c = 0; c < 4; ++c)
					{
						const Key key = lp_key(v[c], 4 * (best_at + u * LP_THREADS + tid) + c - cut);
						if (key != 0 && key >= least) found[atomicAdd(&n_found, 1)] = key;
					}
				}
		}
		__syncthreads();
		// Those threads' groups once more, a warp a thread.
		list = 0;
		for (int w = warp; w < n_again; w += LP_WARPS)
			for (int j0 = v0 + again[w]; j0 < v1; j0 += 32 * LP_THREADS)
			{
				const int j = j0 + lane * LP_THREADS;
				const float4 v4 = j < v1 ? load(j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
				const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
				for (int c = 0; c < 4; ++c)
				{
					Key key = lp_key(v[c], 4 * j + c - cut);
					if (key < least) key = 0;
					if (__any_sync(0xffffffffu, key != 0)) list = lp_merge(list, lp_sort(key, lane), lane);
				}
			}
		if (list != 0) found[atomicAdd(&n_found, 1)] = list;
		__syncthreads();
		if (warp == 0)
		{
			list = 0;
			for (int i = 0; i < n_found; i += 32) list = lp_merge(list, lp_sort(i + lane < n_found ? found[i + lane] : 0, lane), lane);
			mine.top[lane] = list;
		}
	}
	__syncthreads();
	if (tid == 0)
	{
		s = warp_stat[0];
		before = warp_before[0];
		for (int w = 1; w < LP_WARPS; ++w) s = lp_join(s, warp_stat[w], k), before += warp_before[w];
		mine.stat = s;
		mine.before = before;
	}
	__syncthreads();
	if (a.parts > 1) cluster_sync();
	if (part == 0 && warp == 0)
	{
		Key list = TOP ? mine.top[lane] : 0;
		s = mine.stat;
		before = mine.before;
		for (int p = 1; p < a.parts; ++p)
		{
			const Part* other = reinterpret_cast<const Part*>(cluster_map(&mine, p));
			if (TOP) list = lp_merge(list, other->top[lane], lane);
			s = lp_join(s, other->stat, k);
			before += other->before;
		}
		const double lz = log((double)s.z), scale = (double)l.scale;
		if (lane == 0)
		{
			if (l.logprob)
				l.logprob[r] = !in ? 0.0f : s.z == 0.0f ? -INFINITY : (float)(((double)xt - (double)s.m) * scale - lz);
			if (l.rank) l.rank[r] = in ? before : -1;
			if (l.entropy) l.entropy[r] = s.z == 0.0f ? 0.0f : (float)(lz - (double)s.h * 0.69314718055994530942 / (double)s.z);
		}
		if (TOP && lane < l.top)
		{
			if (l.top_ids) l.top_ids[r * l.top + lane] = list ? lp_index(list) : -1;
			if (l.top_logprobs)
				l.top_logprobs[r * l.top + lane] = list ? (float)(((double)lp_value(list) - (double)s.m) * scale - lz) : -INFINITY;
		}
	}
	__syncwarp();
	if (a.parts > 1) cluster_sync(); // nobody reads this CTA's part any more
}

// The CTAs that share a row: the least of the waves that n * parts CTAs make of what the GPU holds at once (two a SM;
// clusters do not fill every SM) times a CTA's time, a row's share and about 4096 logits' worth of start and end.
int lp_parts(long long n, int n_vocab)
{
	static const int slots[] = {296, 296, 284, 264};
	int best = 1;
	double least = 0;
	for (int i = 0, parts = 1; parts <= LP_CLUSTER; ++i, parts *= 2)
	{
		const double t = (double)((n * parts + slots[i] - 1) / slots[i]) * ((double)n_vocab / parts + 4096.0 * (1 + (parts > 1)));
		if (parts == 1 || t < least) least = t, best = parts;
	}
	return best;
}

} // namespace
} // namespace nncu

using namespace nncu;

extern "C" int nncu_logprobs_dev(const nncu_logprobs* l, void* stream)
{
	if (!l) return refuse("logprobs: NULL argument");
	if (l->n < 0 || l->n_vocab <= 0 || l->n_vocab > 1 << 30) return refuse("logprobs: bad n or n_vocab (up to 2^30)");
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
	LpArgs a{*l, (float)fmin((double)l->scale * 1.44269504088896340736, (double)FLT_MAX), lp_parts(l->n, l->n_vocab)};
	cudaLaunchConfig_t cfg{};
	cudaLaunchAttribute at{};
	at.id = cudaLaunchAttributeClusterDimension;
	at.val.clusterDim.x = a.parts, at.val.clusterDim.y = at.val.clusterDim.z = 1;
	cfg.attrs = &at;
	cfg.numAttrs = a.parts > 1;
	cfg.blockDim = dim3(LP_THREADS);
	cfg.stream = static_cast<cudaStream_t>(stream);
	const bool tops = l->top > 0 && (l->top_ids || l->top_logprobs);
	int e = 0;
	const int most = INT32_MAX / LP_CLUSTER; // rows of a launch
	for (long long r0 = 0; r0 < l->n && !e; r0 += most)
	{
		const int rows = (int)(l->n - r0 < most ? l->n - r0 : most);
		cfg.gridDim = dim3((unsigned)rows * a.parts);
		e = (int)(tops ? cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, a) : cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, a));
		note_launches(1);
		a.l.logits += (size_t)rows * a.l.stride;
		if (a.l.tokens) a.l.tokens += rows;
		if (a.l.rank) a.l.rank += rows;
		if (a.l.logprob) a.l.logprob += rows;
		if (a.l.entropy) a.l.entropy += rows;
		if (a.l.top_ids) a.l.top_ids += (size_t)rows * l->top;
		if (a.l.top_logprobs) a.l.top_logprobs += (size_t)rows * l->top;
	}
	if (e) cudaGetLastError();
	return e ? set_cuda_error(e, "logprobs launch") : NNCU_OK;
}
