// k_i8_linear.cu -- the product of 8-bit tokens and weights
// (nncu_i8_linear_dev) on the 5th-generation tensor cores.
//
// Mathematics. y[t][o] = xs[t] ws[o] sum_c x[t][c] w[o][c]: the codes go to
// tcgen05.mma kind::i8 as they are and their sums are exact 32-bit integers,
// so any order of summing, any split over the columns and any tile give the
// same bits; the scales are an epilogue.
//
// Channels are the M dimension (a TMEM lane each), tokens the N dimension (a
// column each), both operands K-major rows of 128 codes, 128-byte swizzled as
// TMA writes them. A thread of the epilogue holds one channel, so a warp's
// store of one token's 32 channels is one 128-byte line.
//
// Few tokens are bound by the weights' bytes (16 x 2560 to 262144 channels: 104
// us, the copy rate) and, where the weights are small, by the chain of launch,
// first copies, stages and epilogue (1 x 4096 to 6144: 6.0 us of 3.8); many by
// the products, the copies out of L2 and the card's power (8192 x 4096 to 6144:
// 140 us, the tensor pipe 80 % busy at 1.66 GHz).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>

#include "i8.h"
#include "i8_plan.h"
#include "tc.cuh"

namespace nncu
{
namespace
{

constexpr int KB = I8_KB, W_BYTES = I8_W_BYTES, MAX_STAGES = I8_MAX_STAGES;

__device__ unsigned g_i8_waits_out; // bounded waits that ran out

struct Args
{
	int n_tok, rows, bn, n_kb, stages, split; // n_kb: stages of the columns
	int panels; // of a stage: one or two
	int tiles_o, tiles_t;
	const float* xs;
	const float* ws;
	const float* bias;
	const float* add;
	float* y;
	size_t add_stride, y_stride;
};

// Instruction descriptor of kind::i8: signed 8-bit operands, both K-major, 32-bit integer sums.
__host__ __device__ constexpr uint32_t i8_idesc(int M, int N)
{
	return (2u << 4) | (1u << 7) | (1u << 10) | (((uint32_t)N >> 3) << 17) | (((uint32_t)M >> 4) << 24);
}

// The products are issued by a whole warp, converged, and executed by its elected lane; conditions on their way are
// votes or go by the launch's own numbers, so that the operands' descriptors live in the warp's uniform registers
// (from a branch that one lane takes, a product cost about 200 cycles, whatever its size).
__device__ __forceinline__ uint32_t elect_one()
{
	uint32_t r;
	asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
	return r;
}
// D (+)= A B, both in shared memory: a, b the low words of their descriptors, `high` the word that they share.
template <int GROUP>
__device__ __forceinline__ void mma_i8(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t id, uint32_t acc, uint32_t lead)
{
	if constexpr (GROUP == 1)
		asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
		             "mov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %3};\n\t"
		             "@q tcgen05.mma.cta_group::1.kind::i8 [%0], x, y, %4, p;\n\t}" ::"r"(d),
		             "r"(a), "r"(b), "r"(high), "r"(id), "r"(acc), "r"(lead)
		             : "memory");
	else
		asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
		             "mov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %3};\n\t"
		             "@q tcgen05.mma.cta_group::2.kind::i8 [%0], x, y, %4, p;\n\t}" ::"r"(d),
		             "r"(a), "r"(b), "r"(high), "r"(id), "r"(acc), "r"(lead)
		             : "memory");
}
// The products so far done: an arrival on the barrier, the pair's on the one at this place of both CTAs.
template <int GROUP>
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t lead, uint16_t both = 0)
{
	if constexpr (GROUP == 1)
		asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
		             "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
		             "r"(lead)
		             : "memory");
	else
		asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
		             "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(
		                 smem_u32(bar)),
		             "r"(lead), "h"(both)
		             : "memory");
}
// The copies are issued the same way. One box of a map into shared memory; in a pair (GROUP 2) the barrier may be the
// other CTA's.
template <int GROUP>
__device__ __forceinline__ void tma2(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint32_t lead)
{
	if constexpr (GROUP == 1)
		asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
		             "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
		             "l"(map), "r"(x), "r"(y), "r"(bar), "r"(lead)
		             : "memory");
	else
		asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
		             "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(
		                 dst),
		             "l"(map), "r"(x), "r"(y), "r"(bar), "r"(lead)
		             : "memory");
}
__device__ __forceinline__ void expect(uint64_t* bar, uint32_t bytes, uint32_t lead)
{
	asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
	             "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
	             "r"(bytes), "r"(lead)
	             : "memory");
}
__device__ __forceinline__ void cluster_sync()
{
	asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of `addr` (this CTA's shared memory) in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank)
{
	uint32_t r;
	asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
	return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int v)
{
	asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar)
{
	asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map)
{
	asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity)
{
	const bool ok = mbar_wait_bounded(bar, parity, nullptr, 0);
	if (!ok) atomicAdd(&g_i8_waits_out, 1u);
	return ok;
}

// A place of the ring of stages and the round that it is in (a division by the number of stages costs as much as a stage).
struct Ring
{
	int s = 0;
	uint32_t round = 0;
	__device__ __forceinline__ void next(int stages)
	{
		if (++s == stages) s = 0, ++round;
	}
};

// After a wait that ran out: what is in flight lands before the CTA ends (the places behind `at`, a round of them).
__device__ __forceinline__ void land(uint64_t* full, Ring at, int stages)
{
	for (int s = 0; s < stages; ++s)
		if (s < at.s || at.round > 0) wait(&full[s], (s < at.s ? at.round : at.round - 1) & 1);
}

__device__ __forceinline__ uint32_t pow2_cols(uint32_t n) { return n <= 32 ? 32 : 1u << (32 - __clz(n - 1)); }

// What `n` tokens from t on have to add to a channel.
template <int C>
__device__ __forceinline__ void get_add(const Args& a, int t, int o, float (&more)[C], int n)
{
	const float* p = a.add + (size_t)t * a.add_stride + o;
#pragma unroll
	for (int c = 0; c < C; ++c, p += a.add_stride) more[c] = c < n ? *p : 0.0f;
}

// A channel's sums of C tokens from t on, scaled and out; `n` of them are real.
template <bool ADD, int C>
__device__ __forceinline__ void put(const Args& a, int t, int o, const int (&acc)[C], const float* xs, float ws, float bias,
                                    const float (&more)[C], int n)
{
	float v[C];
#pragma unroll
	for (int c = 0; c < C; ++c) v[c] = fmaf(__int2float_rn(acc[c]) * xs[c], ws, bias);
	if (ADD)
#pragma unroll
		for (int c = 0; c < C; ++c) v[c] += more[c];
	float* y = a.y + (size_t)t * a.y_stride + o;
	if (n >= C)
	{
#pragma unroll
		for (int c = 0; c < C; ++c, y += a.y_stride) *y = v[c];
	}
	else
	{
#pragma unroll
		for (int c = 0; c < C; ++c, y += a.y_stride)
			if (c < n) *y = v[c];
	}
}

constexpr int THREADS = 320; // a warp for the loads, one for the products, eight for the epilogue (two to a quarter of TMEM)
constexpr int EPI = 256;

// What is added to a tile's tokens from `from` to `to`, of 128 channels, on its way into L2 while its products run
// (read when they are done, 16 tokens at a time, it took longer than they: 4660 x 2560 to 4096 146 us, so 55, 41 with
// nothing to add).
__device__ __forceinline__ void add_ahead(const Args& a, int o0, int t0, int from, int to)
{
	for (int i = (int)threadIdx.x - 64; from + i / 4 < to; i += EPI)
	{
		const int o = o0 + 32 * (i % 4);
		if (o >= a.rows) continue;
		const float* p = a.add + (size_t)(t0 + from + i / 4) * a.add_stride + o;
		asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
		if (reinterpret_cast<uintptr_t>(p) & 127) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + min(31, a.rows - 1 - o)));
	}
}

// Where the columns of a tile are split: CTA `at` of `n` finishes the tile's tokens from at * per on, and every CTA puts
// its sums of them into that one's shared memory ([CTA][token][128 channels] from `base` on), behind its stages, which may
// still be read. One barrier later they are all there, and nobody looks into another CTA any more.
struct Join
{
	uint32_t base;
	int n, at, per, rank0, rank_step; // (CTA i is the cluster's rank0 + i * rank_step)
	__device__ __forceinline__ int from() const { return at * per; }
	__device__ __forceinline__ int to(int real) const { return min(real, from() + per); }
};

// The epilogue of a whole tile from TMEM: this warp's lanes (channels) and its half of the columns, out or, as sums
// only, to the CTAs that join them.
template <bool ADD>
__device__ __forceinline__ void tile_out(const Args& a, uint32_t tmem, int ch, int o, int t0, int real, const float* xs, float ws,
                                         float bias, const Join& join)
{
	const int side = ((int)threadIdx.x - 64) >> 7, quad = (threadIdx.x >> 5) & 3;
	const bool in = o < a.rows, adds = ADD && join.n == 1 && in;
	float next[16] = {}; // (added: a step ahead)
	if (adds && 16 * side < real) get_add(a, t0 + 16 * side, o, next, real - 16 * side);
	for (int c0 = 16 * side; c0 < real; c0 += 32)
	{
		float f[16], more[16];
#pragma unroll
		for (int c = 0; c < 16; ++c) more[c] = next[c];
		if (adds && c0 + 32 < real) get_add(a, t0 + c0 + 32, o, next, real - c0 - 32);
		int v[16];
		tmem_ld16(tmem + ((uint32_t)quad << 21) + c0, f);
		tmem_wait_ld();
#pragma unroll
		for (int c = 0; c < 16; ++c) v[c] = __float_as_int(f[c]);
		if (join.n > 1)
		{
			const uint32_t mine = join.base + (join.at * join.per * 128 + ch) * 4;
			int to = c0 / join.per, i = c0 - to * join.per;
			uint32_t there = mapa(mine, join.rank0 + to * join.rank_step);
#pragma unroll
			for (int c = 0; c < 16; ++c)
			{
				if (i == join.per) i = 0, ++to, there = mapa(mine, join.rank0 + to * join.rank_step);
				st_cluster(there + i++ * 512, v[c]);
			}
		}
		else if (in)
			put<ADD>(a, t0 + c0, o, v, xs + c0, ws, bias, more, real - c0);
	}
}

// The tokens that this CTA joins, from its own shared memory, four channels a lane, a warp a token. `arrive`: the barrier;
// what does not wait for it is read before. `channel`: the channels' scales and biases.
template <bool ADD, class Arrive>
__device__ __forceinline__ void join_out(const Args& a, const Join& join, const int* sums, int o0, int t0, int real, const float* xs,
                                         const float (*channel)[128], Arrive arrive)
{
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, o = o0 + 4 * lane, left = a.rows - o, end = join.to(real);
	float ws[4], bias[4];
#pragma unroll
	for (int j = 0; j < 4; ++j) ws[j] = channel[0][4 * lane + j], bias[j] = channel[1][4 * lane + j];
	const auto in_fours = [&](const float* p, size_t stride) { return left >= 4 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
	const bool wide = in_fours(a.y, a.y_stride), add_wide = ADD && in_fours(a.add, a.add_stride);
	const auto get = [&](int c) {
		const float* p = a.add + (size_t)(t0 + c) * a.add_stride + o;
		if (add_wide) return *reinterpret_cast<const float4*>(p);
		return make_float4(left > 0 ? p[0] : 0.0f, left > 1 ? p[1] : 0.0f, left > 2 ? p[2] : 0.0f, left > 3 ? p[3] : 0.0f);
	};
	int c = join.from() + warp;
	float4 next = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
	if (ADD && c < end) next = get(c);
	__syncwarp();
	arrive();
	for (; c < end; c += THREADS / 32)
	{
		const float4 more = next;
		if (ADD && c + THREADS / 32 < end) next = get(c + THREADS / 32);
		const int4* from = reinterpret_cast<const int4*>(sums + (c - join.from()) * 128) + lane;
		int4 sum = from[0];
#pragma unroll
		for (int i = 1; i < 8; ++i)
			if (i < join.n)
			{
				const int4 q = from[i * join.per * 32];
				sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
			}
		const int acc[4] = {sum.x, sum.y, sum.z, sum.w};
		const float of[4] = {more.x, more.y, more.z, more.w};
		float v[4];
#pragma unroll
		for (int j = 0; j < 4; ++j)
		{
			v[j] = fmaf(__int2float_rn(acc[j]) * xs[c], ws[j], bias[j]);
			if (ADD) v[j] += of[j];
		}
		float* y = a.y + (size_t)(t0 + c) * a.y_stride + o;
		if (wide)
			*reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
		else
#pragma unroll
			for (int j = 0; j < 4; ++j)
				if (j < left) y[j] = v[j];
	}
}

// Channel tiles that are walked together: their weights come from HBM once and the rows of y are written whole.
constexpr int P_GROUP = 32;

// The channels (`wide` a tile) and tokens of tile `id`.
__device__ __forceinline__ void place(const Args& a, int id, int wide, int& o0, int& t0)
{
	if (a.tiles_t == 1)
	{
		o0 = id * wide, t0 = 0;
		return;
	}
	const int per = min(P_GROUP, a.tiles_o) * a.tiles_t, g = id / per, in = id % per;
	const int size = min(P_GROUP, a.tiles_o - g * P_GROUP);
	o0 = (g * P_GROUP + in % size) * wide;
	t0 = in / size * a.bn;
}

// ---- few tokens ------------------------------------------------------------------------
//
// A cluster of `split` CTAs per tile of 128 channels x bn tokens, each with its
// share of the columns; every CTA adds up the sums of a share of the tokens,
// which the others have put into its shared memory (integers: no order).

// (ADD: its code and registers apart; what adds nothing took one to two percent longer with them.)
template <bool ADD>
__global__ void __launch_bounds__(THREADS, 2)
	i8_split_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const Args a)
{
	extern __shared__ uint8_t raw[];
	__shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], done;
	__shared__ uint32_t tmem_slot;
	__shared__ float xs_s[256], channel_s[2][128];
	uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	const int split = a.split, rank = (int)blockIdx.x % split; // (clusters lie along x)
	int o0, t0;
	place(a, (int)(blockIdx.x / split), 128, o0, t0);
	const int k0 = (int)((long long)a.n_kb * rank / split), n = (int)((long long)a.n_kb * (rank + 1) / split) - k0;
	const uint32_t x_at = W_BYTES * a.panels, stage = x_at + a.bn * KB * a.panels, cols = pow2_cols(a.bn);
	const int real = min(a.bn, a.n_tok - t0);
	const Join join{smem_u32(smem) + a.stages * stage, split, rank, (a.bn + split - 1) / split, 0, 1};

	if (threadIdx.x == 0)
	{
		prefetch_map(&wmap);
		prefetch_map(&xmap);
		for (int s = 0; s < a.stages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
		mbar_init(&done, 1);
		fence_barrier_init();
	}
	if (warp == 1) tmem_alloc(&tmem_slot, cols);
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = tmem_slot;
	if (split > 1) cluster_sync(); // all have begun: their memory may be written
	griddep_launch_dependents();
	griddep_wait(); // what came before on the stream is done: up to here nothing was read that it may write

	if (warp == 0)
	{
		const uint32_t lead = elect_one(), base = smem_u32(smem);
		Ring at;
		bool ok = true;
		for (int i = 0; i < n; ++i, at.next(a.stages))
		{
			if (at.round > 0 && !(ok = __all_sync(0xffffffffu, wait(&empty[at.s], (at.round - 1) & 1)))) break;
			expect(&full[at.s], stage, lead);
			const uint32_t dst = base + at.s * stage, bar = smem_u32(&full[at.s]);
			const int k = (k0 + i) * KB * a.panels;
			tma2<1>(dst, &wmap, k, o0, bar, lead);
			tma2<1>(dst + x_at, &xmap, k, t0, bar, lead);
			if (a.panels > 1) // (past the last column: zeros)
			{
				tma2<1>(dst + W_BYTES, &wmap, k + KB, o0, bar, lead);
				tma2<1>(dst + x_at + a.bn * KB, &xmap, k + KB, t0, bar, lead);
			}
		}
		if (!ok) land(full, at, a.stages);
		__syncwarp();
	}
	else if (warp == 1)
	{
		const uint32_t lead = elect_one(), id = i8_idesc(128, a.bn), high = (uint32_t)(sdesc(0, 16, 1024) >> 32);
		const uint32_t base = (uint32_t)sdesc(smem_u32(smem), 16, 1024); // (the stages' addresses stay within its field)
		Ring at;
		for (int i = 0; i < n; ++i, at.next(a.stages))
		{
			if (!__all_sync(0xffffffffu, wait(&full[at.s], at.round & 1))) break;
			tc_fence_after();
			const uint32_t da = base + at.s * (stage >> 4), db = da + (x_at >> 4);
#pragma unroll
			for (int k = 0; k < KB / 32; ++k) mma_i8<1>(tmem, da + 2 * k, db + 2 * k, high, id, i > 0 || k > 0, lead);
			if (a.panels > 1)
#pragma unroll
				for (int k = 0; k < KB / 32; ++k)
					mma_i8<1>(tmem, da + (W_BYTES >> 4) + 2 * k, db + a.bn * (KB >> 4) + 2 * k, high, id, 1, lead);
			commit<1>(&empty[at.s], lead);
			if (i == n - 1) commit<1>(&done, lead);
		}
	}
	else
	{
		const int ch = (warp & 3) * 32 + lane, o = o0 + ch;
		const bool in = o < a.rows;
		const float ws = in ? a.ws[o] : 0.0f, bias = in && a.bias ? a.bias[o] : 0.0f;
		if (split > 1 && warp < 6) channel_s[0][ch] = ws, channel_s[1][ch] = bias;
		for (int c = (int)threadIdx.x - 64; c < a.bn; c += EPI) xs_s[c] = c < real ? a.xs[t0 + c] : 0.0f;
		if (ADD) add_ahead(a, o0, t0, join.from(), join.to(real));
		named_sync(1, EPI);
		const bool ok = wait(&done, 0);
		tc_fence_after();
		if (__all_sync(0xffffffffu, ok)) tile_out<ADD>(a, tmem, ch, o, t0, real, xs_s, ws, bias, join);
		tc_fence_before();
	}
	__syncthreads();
	if (split > 1) join_out<ADD>(a, join, reinterpret_cast<const int*>(smem + a.stages * stage), o0, t0, real, xs_s, channel_s, cluster_sync);
	if (warp == 1)
	{
		tc_fence_after();
		tmem_dealloc(tmem, cols);
	}
}

// ---- many tokens ------------------------------------------------------------------------
//
// One pair of CTAs per two SMs, walking tiles of 256 channels x bn tokens: each
// CTA brings 128 of the channels and half of the tokens, and one product
// (cta_group::2) of both SMs' tensor cores reads both. Two accumulators in TMEM:
// the epilogue of a tile runs beside the next one's products.

template <bool ADD>
__global__ void __launch_bounds__(THREADS, 1)
	i8_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const Args a)
{
	extern __shared__ uint8_t raw[];
	__shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2];
	__shared__ uint32_t tmem_slot;
	__shared__ float xs_s[2][256], channel_s[2][128];
	uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	const int split = a.split, in_cluster = (int)blockIdx.x % (2 * split), rank = in_cluster & 1, first = in_cluster - rank, part = in_cluster >> 1;
	const int pair = (int)blockIdx.x / (2 * split), pairs = (int)gridDim.x / (2 * split); // (clusters, where they are of more)
	const int k0 = (int)((long long)a.n_kb * part / split), n_kb = (int)((long long)a.n_kb * (part + 1) / split) - k0;
	const int tiles = a.tiles_o * a.tiles_t, half = a.bn / 2;
	const uint32_t x_at = W_BYTES * a.panels, stage = x_at + half * KB * a.panels;
	const Join join{smem_u32(smem) + a.stages * stage, split, part, (a.bn + split - 1) / split, rank, 2};

	if (threadIdx.x == 0)
	{
		prefetch_map(&wmap);
		prefetch_map(&xmap);
		for (int s = 0; s < a.stages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
		for (int b = 0; b < 2; ++b) mbar_init(&acc_full[b], 1), mbar_init(&acc_empty[b], 2 * EPI / 32);
		fence_barrier_init();
	}
	if (warp == 1)
	{
		asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u)
		             : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
	}
	tc_fence_before();
	__syncthreads();
	cluster_sync(); // both CTAs' barriers are there
	tc_fence_after();
	constexpr uint32_t tmem = 0; // (512 columns are all there are: the allocation starts at the first)
	griddep_launch_dependents();
	griddep_wait();

	if (warp == 0)
	{
		const uint32_t lead = elect_one(), base = smem_u32(smem);
		Ring at;
		bool ok = true;
		for (int id = pair; id < tiles && ok; id += pairs)
		{
			int o0, t0;
			place(a, id, 256, o0, t0);
			for (int k = 0; k < n_kb; ++k, at.next(a.stages))
			{
				if (at.round > 0 && !(ok = __all_sync(0xffffffffu, wait(&empty[at.s], (at.round - 1) & 1)))) break;
				if (rank == 0) expect(&full[at.s], 2 * stage, lead); // both CTAs' bytes land on the first one's barrier
				const uint32_t dst = base + at.s * stage, bar = mapa(smem_u32(&full[at.s]), first);
				const int c = (k0 + k) * KB * a.panels;
				tma2<2>(dst, &wmap, c, o0 + rank * 128, bar, lead);
				tma2<2>(dst + x_at, &xmap, c, t0 + rank * half, bar, lead);
				if (a.panels > 1)
				{
					tma2<2>(dst + W_BYTES, &wmap, c + KB, o0 + rank * 128, bar, lead);
					tma2<2>(dst + x_at + half * KB, &xmap, c + KB, t0 + rank * half, bar, lead);
				}
			}
		}
		if (!ok && rank == 0) land(full, at, a.stages);
		__syncwarp();
	}
	else if (warp == 1)
	{
		if (rank == 0)
		{
			const uint32_t lead = elect_one(), idesc = i8_idesc(256, a.bn), high = (uint32_t)(sdesc(0, 16, 1024) >> 32);
			const uint16_t both = (uint16_t)(3u << first);
			const uint32_t base = (uint32_t)sdesc(smem_u32(smem), 16, 1024); // (the stages' addresses stay within its field)
			Ring at;
			int n = 0;
			bool ok = true;
			for (int id = pair; id < tiles && ok; id += pairs, ++n)
			{
				const int b = n & 1;
				if (n >= 2 && !(ok = __all_sync(0xffffffffu, wait(&acc_empty[b], (uint32_t)(n / 2 - 1) & 1)))) break;
				tc_fence_after();
				for (int k = 0; k < n_kb; ++k, at.next(a.stages))
				{
					if (!(ok = __all_sync(0xffffffffu, wait(&full[at.s], at.round & 1)))) break;
					tc_fence_after();
					const uint32_t da = base + at.s * (stage >> 4), db = da + (x_at >> 4);
#pragma unroll
					for (int q = 0; q < KB / 32; ++q) mma_i8<2>(tmem + b * 256, da + 2 * q, db + 2 * q, high, idesc, k > 0 || q > 0, lead);
					if (a.panels > 1)
#pragma unroll
						for (int q = 0; q < KB / 32; ++q)
							mma_i8<2>(tmem + b * 256, da + (W_BYTES >> 4) + 2 * q, db + half * (KB >> 4) + 2 * q, high, idesc, 1, lead);
					commit<2>(&empty[at.s], lead, both);
					if (k == n_kb - 1) commit<2>(&acc_full[b], lead, both);
				}
			}
		}
	}
	else
	{
		const int ch = (warp & 3) * 32 + lane;
		int n = 0;
		bool ok = true; // (after a wait that ran out the warp goes on through the barriers, without work)
		const auto ahead = [&](int id) {
			if (!ADD || id >= tiles) return;
			int o0, t0;
			place(a, id, 256, o0, t0);
			add_ahead(a, o0 + rank * 128, t0, join.from(), join.to(min(a.bn, a.n_tok - t0)));
		};
		ahead(pair);
		for (int id = pair; id < tiles; id += pairs, ++n)
		{
			const int b = n & 1;
			int o0, t0;
			place(a, id, 256, o0, t0);
			ahead(id + pairs);
			const int o = o0 + rank * 128 + ch, real = min(a.bn, a.n_tok - t0);
			const bool in = o < a.rows;
			const float ws = in ? a.ws[o] : 0.0f, bias = in && a.bias ? a.bias[o] : 0.0f;
			if (split > 1 && warp < 6) channel_s[0][ch] = ws, channel_s[1][ch] = bias;
			// (a warp is at most one tile behind another: the barrier below lets none two ahead)
			for (int c = (int)threadIdx.x - 64; c < a.bn; c += EPI) xs_s[b][c] = c < real ? a.xs[t0 + c] : 0.0f;
			named_sync(1, EPI);
			ok = __all_sync(0xffffffffu, ok && wait(&acc_full[b], (uint32_t)(n / 2) & 1));
			if (!ok) continue;
			tc_fence_after();
			tile_out<ADD>(a, tmem + b * 256, ch, o, t0, real, xs_s[b], ws, bias, join);
			tc_fence_before();
			__syncwarp();
			if (lane == 0) arrive_cluster(mapa(smem_u32(&acc_empty[b]), first));
		}
	}
	__syncthreads();
	// (the barrier also for this: the other CTA's products read this one's memory, its epilogue arrives here)
	if (split > 1) // (one tile a cluster)
	{
		int o0, t0;
		place(a, pair, 256, o0, t0);
		join_out<ADD>(a, join, reinterpret_cast<const int*>(smem + a.stages * stage), o0 + rank * 128, t0, min(a.bn, a.n_tok - t0), xs_s[0], channel_s, cluster_sync);
	}
	else
		cluster_sync();
	if (warp == 1)
	{
		tc_fence_after();
		asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
	}
}

// ---- host ----------------------------------------------------------------------------------

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, looked up through the runtime (the library loads without the driver).
Encode encoder()
{
	static const Encode e = [] {
		void* fn = nullptr;
		cudaDriverEntryPointQueryResult q;
		if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
		    q != cudaDriverEntryPointSuccess)
			fn = nullptr;
		return reinterpret_cast<Encode>(fn);
	}();
	return e;
}

// A map over n rows of `cols` codes, boxes of 128 codes x box rows, swizzled; past the edges it reads zeros.
bool code_map(CUtensorMap* map, const int8_t* p, int n, int cols, size_t stride, int box)
{
	const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)n};
	const cuuint64_t strides[1] = {n > 1 ? (cuuint64_t)stride : ((cuuint64_t)cols + 15) / 16 * 16};
	const cuuint32_t boxes[2] = {KB, (cuuint32_t)box}, estr[2] = {1, 1};
	const Encode e = encoder();
	return e && e(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, boxes, estr,
	              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
	              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int configure()
{
	static bool configured[64] = {};
	int dev = 0;
	cudaError_t ce = cudaGetDevice(&dev);
	if (ce != cudaSuccess) return (int)ce;
	if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
	if (configured[dev]) return 0;
	for (const auto kernel : {i8_split_kernel<false>, i8_split_kernel<true>, i8_pair_kernel<false>, i8_pair_kernel<true>})
	{
		ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, I8_SMEM_MOST);
		if (ce != cudaSuccess) return (int)ce;
	}
	configured[dev] = true;
	return 0;
}

} // namespace

int launch_i8_linear(const nncu_i8_linear& l, void* stream)
{
	int e = configure();
	if (e) return e;
	Args a{};
	a.n_tok = l.n_tok, a.rows = l.rows;
	a.xs = l.x_scales, a.ws = l.w_scales, a.bias = l.bias, a.add = l.add, a.y = l.y;
	a.add_stride = l.add_stride, a.y_stride = l.y_stride;
	const I8Plan p = i8_plan(l.n_tok, l.rows, l.cols);
	a.bn = p.bn, a.split = p.split, a.panels = p.panels, a.n_kb = (l.cols + KB * p.panels - 1) / (KB * p.panels);
	a.stages = i8_stages(p);
	CUtensorMap xm, wm;
	if (!code_map(&xm, l.x, l.n_tok, l.cols, l.x_stride, p.pair ? p.bn / 2 : p.bn) ||
	    !code_map(&wm, l.w, l.rows, l.cols, l.w_stride, 128))
		return (int)cudaErrorInvalidValue;
	a.tiles_o = p.tiles_o, a.tiles_t = p.tiles_t;
	cudaLaunchAttribute at[2]{};
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	at[1].id = cudaLaunchAttributeClusterDimension;
	at[1].val.clusterDim.x = (p.pair ? 2 : 1) * p.split, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
	cudaLaunchConfig_t cfg{};
	cfg.stream = static_cast<cudaStream_t>(stream);
	cfg.attrs = at;
	cfg.numAttrs = at[1].val.clusterDim.x > 1 ? 2 : 1;
	cfg.blockDim = dim3(THREADS);
	cfg.dynamicSmemBytes = i8_smem(p);
	const long long tiles = (long long)p.tiles_o * p.tiles_t;
	if (p.pair)
	{
		cfg.gridDim = dim3(2 * (unsigned)(p.split > 1 ? tiles * p.split : min(tiles, (long long)I8_SMS / 2)));
		return (int)cudaLaunchKernelEx(&cfg, l.add ? i8_pair_kernel<true> : i8_pair_kernel<false>, xm, wm, a);
	}
	cfg.gridDim = dim3((unsigned)(tiles * p.split));
	return (int)cudaLaunchKernelEx(&cfg, l.add ? i8_split_kernel<true> : i8_split_kernel<false>, xm, wm, a);
}

int i8_waits_out(unsigned* count, void* stream)
{
	const auto st = static_cast<cudaStream_t>(stream);
	cudaError_t ce = cudaMemcpyFromSymbolAsync(count, g_i8_waits_out, sizeof *count, 0, cudaMemcpyDeviceToHost, st);
	if (ce == cudaSuccess) ce = cudaStreamSynchronize(st);
	return (int)ce;
}

} // namespace nncu
