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
// logit and the largest outside of that one's group. The top-th of the warps'
// first four bounds the answer from below; what passes it lies with about `top`
// threads, nearly always in the group of 16 that each reads again, in the rest of
// a thread's share only where its second group passes the bound too. Where too
// much passes (equal logits, few warps with any), the top-th of all threads'
// largest is the bound, which `top` threads pass (64 x 151936, all equal: 50 us).
//
// Bound by memory where rows are many (2047 x 128256: 159 us, the copy rate); a
// row is shared by up to eight CTAs (a cluster, whose parts meet in the first
// one's shared memory) where they are few: 64 x 151936 with 5 alternatives 13.3
// us (the copy rate: 5.9), 1 x 262144 with 20 8.0 us. Their ends are short chains:
// the largest first (redux), then sums; every warp's parts straight to the first
// CTA; a thread's group read again while its sums are joined; runs merged by
// counting (14.4 and 8.9 us with pairwise joins and bitonic merges of the parts).
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "logprobs_plan.h"
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
__device__ __forceinline__ void* cluster_map(const void* p, int rank)
{
	uint64_t r;
	asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
	return reinterpret_cast<void*>(r);
}

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

constexpr int LP_TOP = 32;
constexpr int LP_ITEMS = 4;   // 16-byte loads a thread has in flight
constexpr int LP_FIRST = 4;   // of each warp's candidates, those that bound the others

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

__device__ __forceinline__ float lp_max(float x)
{
	float m;
	asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
	return m;
}

// What a part of a row knows of its softmax, in base 2: the largest logit, the sum of e = 2^((x - m) k) and that of e
// times its exponent.
struct Stat
{
	float m, z, h;
};
// A warp's parts as one, in every lane: first the largest logit, then sums.
__device__ __forceinline__ Stat lp_join(Stat s, float k)
{
	const float m = lp_max(s.m);
	const float d = fmaxf((s.m - m) * k, -1e5f), c = ex2(d); // (held above -infinity, so that an empty part adds zeros)
	s.h = c * (s.h + d * s.z);
	s.z *= c;
	s.m = m;
#pragma unroll
	for (int i = 16; i > 0; i >>= 1) s.z += __shfl_xor_sync(0xffffffffu, s.z, i), s.h += __shfl_xor_sync(0xffffffffu, s.h, i);
	return s;
}

struct LpArgs
{
	nncu_logprobs l;
	float k; // scale / ln 2
	int parts; // CTAs that share a row
};

// A row's share of one CTA, in vectors of four logits that lie on 16 bytes: the row's first and last one may be cut.
// (Ordinary loads: the kernel before this one may still write the logits when this one begins, so that they are not
// read-only for its life, which a non-coherent load asks for.)
struct Share
{
	const float* x;
	int n, cut, nvec, v0, v1;
	__device__ __forceinline__ Share(const nncu_logprobs& l, size_t r, int part, int parts) : x(l.logits + r * l.stride), n(l.n_vocab)
	{
		cut = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
		nvec = (n + cut + 3) / 4;
		const int each = (nvec + parts - 1) / parts;
		v0 = min(nvec, part * each), v1 = min(nvec, v0 + each);
	}
	__device__ __forceinline__ const float4* at(int j) const { return reinterpret_cast<const float4*>(x - cut) + j; }
	__device__ __forceinline__ bool whole(int j) const { return j > 0 && j < nvec - 1 && j < v1; }
	__device__ __forceinline__ int index(int j, int c) const { return 4 * j + c - cut; }
	// what is not the share's reads as masked
	__device__ __forceinline__ float4 load(int j) const
	{
		if (whole(j)) return *at(j);
		float v[4];
#pragma unroll
		for (int c = 0; c < 4; ++c)
		{
			const int i = index(j, c);
			v[c] = j < v1 && i >= 0 && i < n ? x[i] : -INFINITY;
		}
		return make_float4(v[0], v[1], v[2], v[3]);
	}
	// the thread's logits of the group of T * LP_ITEMS vectors from g on
	template <int T>
	__device__ __forceinline__ void read(int g, float (&v)[4 * LP_ITEMS]) const
	{
		if (g > 0 && g + T * LP_ITEMS < nvec && g + T * LP_ITEMS <= v1)
		{
#pragma unroll
			for (int u = 0; u < LP_ITEMS; ++u)
			{
				const float4 q = *at(g + u * T + (int)threadIdx.x);
				v[4 * u] = q.x, v[4 * u + 1] = q.y, v[4 * u + 2] = q.z, v[4 * u + 3] = q.w;
			}
		}
		else
#pragma unroll
			for (int u = 0; u < LP_ITEMS; ++u)
			{
				const float4 q = load(g + u * T + (int)threadIdx.x);
				v[4 * u] = q.x, v[4 * u + 1] = q.y, v[4 * u + 2] = q.z, v[4 * u + 3] = q.w;
			}
	}
};

// A thread's largest logits of its share: what the selection goes by.
struct Best
{
	float value, second; // of all groups; of the groups but the one that reached the largest first
	int group;
};

template <int T>
struct Found
{
	static constexpr int WARPS = T / 32, MOST = LP_TOP * 4 * LP_ITEMS + WARPS * LP_TOP;
	Key keys[MOST], lists[WARPS][LP_TOP];
	float bound[WARPS * LP_FIRST], least;
	int n, n_again;
	short again[T];
};

// The likeliest tokens of the CTA's share into out[LP_TOP], falling (0: none); v: the thread's logits of its best group.
template <int T>
__device__ __forceinline__ void lp_select(const Share& sh, const Best& b, const float (&v)[4 * LP_ITEMS], int top, Found<T>& f, Key* out)
{
	constexpr int WARPS = Found<T>::WARPS, MOST = Found<T>::MOST, BOUNDS = WARPS * LP_FIRST;
	const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const auto index = [&](int i) { return sh.index(b.group + (i / 4) * T + tid, i % 4); };
	// The warp's first few of its threads' largest, one after another.
	float left = b.value;
#pragma unroll
	for (int i = 0; i < LP_FIRST; ++i)
	{
		const float m = lp_max(left);
		const uint32_t with = __ballot_sync(0xffffffffu, left == m);
		if (lane == __ffs(with) - 1) left = -INFINITY;
		if (lane == 0) f.bound[warp * LP_FIRST + i] = m;
	}
	if (tid == 0) f.n = f.n_again = 0, f.least = -INFINITY;
	if (tid < LP_TOP) out[tid] = 0;
	__syncthreads();
	// The top-th of them is a bound: that many logits are not below it. Eight threads count for each.
	{
		static_assert(T == 8 * BOUNDS, "eight threads a bound");
		const float x = f.bound[tid / 8];
		int n = 0; // those above x, and in the upper half those not below it
#pragma unroll
		for (int j = tid % 8; j < BOUNDS; j += 8) n += (f.bound[j] > x) + ((f.bound[j] >= x) << 16);
#pragma unroll
		for (int d = 4; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
		if (x > -INFINITY && (n & 0xFFFF) < top && (n >> 16) >= top) f.least = x; // (equal ones write the same)
	}
	__syncthreads();
	// What is not below it lies with the threads whose largest is not, nearly always in that one's group.
	const auto push = [&](Key k) {
		const int i = atomicAdd(&f.n, 1);
		if (i < MOST) f.keys[i] = k;
	};
	const auto give = [&](float low, Key least) {
		if (low == -INFINITY ? b.second > low : b.second >= low) // more may lie in the thread's other groups
		{
			f.again[atomicAdd(&f.n_again, 1)] = (short)tid;
			return;
		}
		uint32_t those = 0;
#pragma unroll
		for (int i = 0; i < 4 * LP_ITEMS; ++i) those |= (v[i] >= low && v[i] > -INFINITY ? 1u : 0u) << i;
		if ((those & (those - 1)) == 0) // one: the largest
		{
			const int i = __ffs(those) - 1;
			const Key k = lp_key(b.value, index(i));
			if (k >= least) push(k);
			return;
		}
#pragma unroll
		for (int i = 0; i < 4 * LP_ITEMS; ++i)
			if (those >> i & 1)
			{
				const Key k = lp_key(v[i], index(i));
				if (k >= least) push(k);
			}
	};
	const float low = f.least;
	if (b.value > -INFINITY && b.value >= low) give(low, 0);
	__syncthreads();
	for (int w = warp; w < f.n_again; w += WARPS) // those threads' vectors once more, a warp a thread
		for (int j = sh.v0 + f.again[w] + lane * T; j < sh.v1; j += 32 * T)
		{
			const float4 q = sh.load(j);
			const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
			for (int c = 0; c < 4; ++c)
				if (e[c] >= low && e[c] > -INFINITY) push(lp_key(e[c], sh.index(j, c)));
		}
	__syncthreads();
	if (f.n > MOST)
	{
		// Too many: few warps hold the largest, or most of the row is equal. The top-th of all threads' firsts (by value and
		// index) bounds the owners to `top` of them, and a warp's list what it takes of each.
		int at = 0; // (the first of the largest, in the group that reached them first)
#pragma unroll
		for (int i = 4 * LP_ITEMS - 1; i >= 0; --i)
			if (v[i] == b.value) at = (i / 4) * 4 * T + i % 4;
		const Key first = lp_key(b.value, sh.index(b.group + tid, 0) + at); // (0 where all are masked)
		Key list = lp_sort(first, lane);
		f.lists[warp][lane] = list;
		__syncthreads();
		for (int d = WARPS / 2; d > 0; d /= 2)
		{
			if (warp < d) f.lists[warp][lane] = list = lp_merge(list, f.lists[warp + d][lane], lane);
			__syncthreads();
		}
		const Key least = f.lists[0][top - 1];
		if (tid == 0) f.n = f.n_again = 0;
		__syncthreads();
		if (first != 0 && first >= least) give(least ? lp_value(least) : -INFINITY, least);
		__syncthreads();
		list = 0;
		for (int w = warp; w < f.n_again; w += WARPS)
			for (int j0 = sh.v0 + f.again[w]; j0 < sh.v1; j0 += 32 * T)
			{
				const float4 q = sh.load(j0 + lane * T);
				const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
				for (int c = 0; c < 4; ++c)
				{
					Key k = lp_key(e[c], sh.index(j0 + lane * T, c));
					if (k < least) k = 0;
					if (__any_sync(0xffffffffu, k != 0)) list = lp_merge(list, lp_sort(k, lane), lane);
				}
			}
		if (list != 0) push(list);
		__syncthreads();
	}
	const int n = f.n;
	for (int i = tid; i < n; i += T)
	{
		const Key k = f.keys[i];
		int above = 0;
#pragma unroll 4
		for (int j = 0; j < n; ++j) above += f.keys[j] > k;
		if (above < LP_TOP) out[above] = k;
	}
}

// What the CTAs that share a row know of it, in the first one's shared memory.
template <bool TOP, int T>
struct Row
{
	Stat stat[LP_CLUSTER][T / 32];
	int before[LP_CLUSTER][T / 32];
	Key top[TOP ? LP_CLUSTER : 1][LP_TOP], all[LP_TOP];
	float m;
	double lz;
};

// The falling runs of `parts` CTAs into one (all: zeros before), each key at the number of keys above it.
template <class R>
__device__ __forceinline__ void lp_merge_parts(R& row, int parts, int lane, int warp)
{
	if (warp >= parts) return;
	const Key k = row.top[warp][lane];
	int above[LP_CLUSTER] = {};
#pragma unroll
	for (int d = 16; d > 0; d >>= 1)
#pragma unroll
		for (int p = 0; p < LP_CLUSTER; ++p) above[p] += row.top[p][above[p] + d - 1] > k ? d : 0; // (past `parts`: not used)
	int n = 0;
#pragma unroll
	for (int p = 0; p < LP_CLUSTER; ++p)
		if (p < parts) n += above[p] + (row.top[p][above[p]] > k); // (all 32 may be above)
	if (k != 0 && n < LP_TOP) row.all[n] = k;
}

template <bool TOP, int T, bool AHEAD>
__global__ void __launch_bounds__(T, lp_ctas(T, AHEAD)) logprobs_kernel(const LpArgs a)
{
	constexpr int WARPS = T / 32, GROUP = T * LP_ITEMS; // vectors (of four logits) that the CTA takes at a time
	static_assert(WARPS >= LP_CLUSTER && WARPS <= 32, "a warp a part, a lane a warp");
	__shared__ Row<TOP, T> row;
	__shared__ std::conditional_t<TOP, Found<T>, int> found;
	const nncu_logprobs& l = a.l;
	const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int part = (int)(blockIdx.x % a.parts);
	const size_t r = blockIdx.x / a.parts;
	const float k = a.k;
	griddep_launch_dependents();
	if (a.parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); // (its end is waited for below: all have begun)
	griddep_wait();

	const Share sh(l, r, part, a.parts);
	float v[4 * LP_ITEMS];
	sh.template read<T>(sh.v0, v); // (before the token's own logit, which waits for two loads in a row)
	const int n = l.n_vocab, tok = l.tokens ? l.tokens[r] : -1;
	const bool in = tok >= 0 && tok < n;
	const float xt = in ? sh.x[tok] : 0.0f;
	const bool hidden = in && !(xt > -INFINITY);   // (a NaN comes as -infinity)
	// What a logit before the token has to pass to come before it (x >= xt is x > the value below xt), and one after it. Of
	// a masked token all that are before it come first: they are counted at the end.
	const float pass = hidden ? INFINITY : nextafterf(xt, -INFINITY), pass_after = hidden ? -INFINITY : xt;
	const int tok_vec = in ? (tok + sh.cut) / 4 : -1;
	Stat s{-FLT_MAX, 0.0f, 0.0f};
	int before = 0;
	Best best{-INFINITY, -INFINITY, sh.v0};
	// AHEAD: the next group's loads are in flight while one is counted (wide, 64 x 151936 top 5: 13.2 us, without 13.7;
	// narrow, 450 x 43807 17.4, without 20.7). The registers for it cost the fifth narrow CTA of an SM (700 x 43807: 29.1 us,
	// five without it 23.7).
	float next[4 * LP_ITEMS];
	for (int g = sh.v0; g < sh.v1;)
	{
		if (AHEAD && g + GROUP < sh.v1) sh.template read<T>(g + GROUP, next);
		float top = -INFINITY;
#pragma unroll
		for (int i = 0; i < 4 * LP_ITEMS; ++i) top = fmaxf(top, v[i]);
		if (TOP)
		{
			if (top > best.value)
				best.second = best.value, best.value = top, best.group = g;
			else
				best.second = fmaxf(best.second, top);
		}
		if (top > s.m)
		{
			const float d = fmaxf((s.m - top) * k, -1e5f), c = ex2(d);
			s.h = c * (s.h + d * s.z);
			s.z *= c;
			s.m = top;
		}
		float2 z = make_float2(0.0f, 0.0f), h = z;
#pragma unroll
		for (int u = 0; u < LP_ITEMS; ++u)
		{
			const float over = g + u * T + tid < tok_vec ? pass : pass_after;
#pragma unroll
			for (int c = 0; c < 4; c += 2)
			{
				const float2 x = make_float2(v[4 * u + c], v[4 * u + c + 1]);
				float2 t = add2(x, make_float2(-s.m, -s.m));
				t = make_float2(t.x * k, t.y * k);
				const float2 e = make_float2(ex2(t.x), ex2(t.y));
				z = add2(z, e);
				h = fma2(e, make_float2(fmaxf(t.x, -200.0f), fmaxf(t.y, -200.0f)), h); // (2^-200 is 0: what is masked adds no 0 * infinity)
				before += x.x > over;
				before += x.y > over;
			}
		}
		s.z += z.x + z.y;
		s.h += h.x + h.y;
		g += GROUP;
		if (AHEAD)
#pragma unroll
			for (int i = 0; i < 4 * LP_ITEMS; ++i) v[i] = next[i];
		else if (g < sh.v1)
			sh.template read<T>(g, v);
	}
	if (in && tid == 0)
	{
		const int v_first = max(0, 4 * tok_vec - sh.cut); // the first of the token's own vector
		if (tok_vec >= sh.v0 && tok_vec < sh.v1) // those before it there: equal, or masked as it is
			for (int i = v_first; i < tok; ++i) before += hidden ? !(sh.x[i] > -INFINITY) : sh.x[i] == xt;
		if (hidden) before += max(0, min(v_first, 4 * sh.v1 - sh.cut) - max(0, 4 * sh.v0 - sh.cut));
	}

	if constexpr (TOP) sh.template read<T>(best.group, v); // (for the selection, while the sums are joined)
	s = lp_join(s, k);
	before = __reduce_add_sync(0xffffffffu, before);
	if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); // (the first CTA has begun)
	Row<TOP, T>& to = a.parts > 1 ? *static_cast<Row<TOP, T>*>(cluster_map(&row, 0)) : row;
	if (lane == 0) to.stat[part][warp] = s, to.before[part][warp] = before;
	if constexpr (TOP)
	{
		if (warp == 0) row.all[lane] = 0;
		lp_select(sh, best, v, l.top, found, a.parts > 1 ? to.top[part] : row.all);
	}
	__syncthreads();
	if (a.parts > 1)
	{
		cluster_sync();
		if (part != 0) return;
		if constexpr (TOP) lp_merge_parts(row, a.parts, lane, warp);
	}
	if (warp == WARPS - 1) // (the last one: the first ones merge)
	{
		s = Stat{-FLT_MAX, 0.0f, 0.0f}, before = 0;
		if (lane < WARPS)
		{
			Stat of[LP_CLUSTER];
#pragma unroll
			for (int p = 0; p < LP_CLUSTER; ++p)
			{
				of[p] = p < a.parts ? row.stat[p][lane] : Stat{-FLT_MAX, 0.0f, 0.0f};
				s.m = fmaxf(s.m, of[p].m);
				before += p < a.parts ? row.before[p][lane] : 0;
			}
#pragma unroll
			for (int p = 0; p < LP_CLUSTER; ++p)
			{
				const float d = fmaxf((of[p].m - s.m) * k, -1e5f), c = ex2(d);
				s.z += c * of[p].z;
				s.h += c * (of[p].h + d * of[p].z);
			}
		}
		s = lp_join(s, k);
		before = __reduce_add_sync(0xffffffffu, before);
		const double lz = log((double)s.z);
		if (lane == 0)
		{
			row.m = s.m, row.lz = lz;
			if (l.logprob) l.logprob[r] = !in ? 0.0f : s.z == 0.0f ? -INFINITY : (float)(((double)xt - (double)s.m) * (double)l.scale - lz);
			if (l.rank) l.rank[r] = in ? before : -1;
			if (l.entropy) l.entropy[r] = s.z == 0.0f ? 0.0f : (float)(lz - (double)s.h * 0.69314718055994530942 / (double)s.z);
		}
	}
	if constexpr (TOP)
	{
		__syncthreads();
		if (tid < l.top)
		{
			const Key key = row.all[tid];
			if (l.top_ids) l.top_ids[r * l.top + tid] = key ? lp_index(key) : -1;
			if (l.top_logprobs)
				l.top_logprobs[r * l.top + tid] = key ? (float)(((double)lp_value(key) - (double)row.m) * (double)l.scale - row.lz) : -INFINITY;
		}
	}
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
	const bool tops = l->top > 0 && (l->top_ids || l->top_logprobs);
	const int rc = check_current_device({l->logits, l->tokens, l->logprob, l->rank, l->entropy, tops ? l->top_ids : nullptr,
	                                     tops ? l->top_logprobs : nullptr},
	                                    "logprobs");
	if (rc != NNCU_OK) return rc;
	LpArgs a{*l, (float)fmin((double)l->scale * 1.44269504088896340736, (double)FLT_MAX), 1};
	const LpPlan plan = lp_plan(l->n, l->n_vocab, tops);
	a.parts = plan.parts;
	cudaLaunchAttribute at[2]{};
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	at[1].id = cudaLaunchAttributeClusterDimension;
	at[1].val.clusterDim.x = a.parts, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
	cudaLaunchConfig_t cfg{};
	cfg.attrs = at;
	cfg.numAttrs = a.parts > 1 ? 2 : 1;
	cfg.blockDim = dim3(plan.wide ? LP_WIDE : LP_NARROW);
	cfg.stream = static_cast<cudaStream_t>(stream);
	const long long most = INT32_MAX / LP_CLUSTER; // rows of a launch
	int e = 0;
	for (long long left = l->n; left > 0 && !e; left -= most)
	{
		const long long rows = left < most ? left : most;
		cfg.gridDim = dim3((unsigned)(rows * a.parts));
		const auto kernel = plan.wide    ? (tops ? logprobs_kernel<true, LP_WIDE, true> : logprobs_kernel<false, LP_WIDE, true>)
		                    : plan.ahead ? (tops ? logprobs_kernel<true, LP_NARROW, true> : logprobs_kernel<false, LP_NARROW, true>)
		                                 : (tops ? logprobs_kernel<true, LP_NARROW, false> : logprobs_kernel<false, LP_NARROW, false>);
		e = (int)cudaLaunchKernelEx(&cfg, kernel, a);
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
