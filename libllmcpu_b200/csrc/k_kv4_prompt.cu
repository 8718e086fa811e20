// k_kv4_prompt.cu -- attention over the paged 4-bit cache for requests with
// many query rows (prompts, chunks of prompts), on the 5th-generation tensor
// cores. (Few rows: k_kv4_attn.cu.)
//
// Work. A block is (request, KV head, 128 NQ query rows; a row is token x
// grouped head, so the heads that share a KV head share its keys' unpacking).
// A block's keys are walked in tiles of 64. A planning kernel (one CTA) lists
// the blocks of the requests from their lengths on the device, cuts those
// with long spans into pieces of about half an SM's share, and the attention
// kernel takes one (piece, KV head) per CTA. Pieces of one block meet in the
// workspace; the last one joins them in order.
//
// Mathematics. 8 bits of scale times 4 of code are exact in a 16-bit float, so
// K and V go to the tensor cores as they are; q and the softmax weights go as
// two 16-bit halves each (22 bits), accumulated in 32:
//
//   S  = Qhi K^T + Qlo K^T   tcgen05.mma, M 128 x N 64, operands in shared memory
//   O += Phi V  + Plo V      tcgen05.mma, M 128 x N D, P from TMEM over its own S
//
// which is twice a 16-bit attention's products for 32-bit results. A row's q
// is scaled by a power of two to fill the 16-bit range, undone in the softmax;
// weights are taken against a held score, 2^11 at it, that moves only when a
// score passes it by 2^4.
//
// Roles (512 threads): warp 0 brings the pages' codes and scales (bulk copies
// into a ring of half tiles: K of tile u, V of tile u - 1, ...); warp 1 owns
// TMEM and issues the products; warps 4-7 unpack half tiles into 16-bit
// operands (128-byte swizzled); warps 8-11 and 12-15 do the softmax of Q tile
// A and B, one row a thread, and write the output. Two S buffers a Q tile: the
// softmax of tile u + 1 runs while P V of tile u and S of tile u + 2 are
// computed. Every wait is bounded; after one that ran out the CTA records an
// error and steps through without waiting.
//
// What bounds it: the products, which take 120 cycles each beside the
// unpacking where they take 53 alone, and (head_dim 256, 128 rows a block) the
// unpacking itself. Six prompts of 200 to 2048 tokens over 777 to 4096 keys,
// 32/8 heads x 128: 571 us, 211 TFLOP/s (422 of 16-bit products); 1000 tokens
// over 16000 keys, 8/4 x 256: 621 us, 204 TFLOP/s.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cfloat>
#include <type_traits>

#include "kv4.cuh"
#include "kv4_plan.h"
#include "tc.cuh"

namespace nncu
{
namespace
{

constexpr int BN = 64;           // keys a tile
constexpr int PT = 512;          // threads
constexpr float HELD = 11.0f, HELD_TOP = 15.0f; // see k_kv4_attn.cu
constexpr int PLAN_THREADS = 1024;
// Each product cuts the accumulator off at 24 bits, always towards zero: over
// a long run of tiles that adds up (6e-6 of the output after 50 tiles). So O
// starts anew every FRESH tiles, and the threads add up what it held, rounded
// to nearest, in a place of the workspace that a CTA takes for itself while it
// runs. There are at least as many places as SMs, and a CTA fills an SM (its
// registers, its tensor memory), so one is always free.
constexpr int FRESH = 6, PLACES = 192, PLACE_TRIES = 1 << 20;

template <int D>
struct PShape
{
	static constexpr int U = D / KV4_GROUP, NQ = D == 256 ? 1 : 2, BR = 128 * NQ, PANELS = D / 64;
	static constexpr int Q_PANEL = 128 * 128, Q_HALF = PANELS * Q_PANEL; // 128 rows x 64 values; one 16-bit half of a Q tile
	static constexpr int KV_PANEL = BN * 128, KV_TILE = PANELS * KV_PANEL;
	static constexpr int KS = D == 256 ? 1 : 2; // unpacked K tiles, and V tiles
	static constexpr int CODES = BN * D / 2, SCALES = BN * U * 2, RAW = CODES + SCALES, RAW_STAGES = D == 256 ? 3 : 4;
	static constexpr int SM_Q = 0, SM_K = SM_Q + NQ * 2 * Q_HALF, SM_V = SM_K + KS * KV_TILE;
	static constexpr int SM_RAW = SM_V + KS * KV_TILE, SM_BAR = SM_RAW + RAW_STAGES * RAW;
	static constexpr int SMEM = SM_BAR + 512 + 1024;
	static_assert(SMEM <= 227 * 1024 && SM_BAR % 16 == 0 && RAW % 16 == 0, "shared memory");
	// TMEM: S of Q tile X, buffer b at 128 X + 64 b (its P: 32 columns of high halves, 32 of low), O behind
	static constexpr uint32_t T_O = NQ * 128, COLS = 512;
	static_assert(NQ * (128 + D) <= 512, "TMEM");
	static constexpr size_t PART = (size_t)BR * (D + 2); // floats a partial result: [D / 4][BR] of 4, then [BR] of 2
};

// A run of a block's key tiles, as the planning kernel lists it.
struct Piece
{
	int r, row0;        // request, first row of the block
	int tile0, tiles;   // of the piece
	int first, n;       // first piece of the block, its number of pieces
	int block, split0;  // the block (its counter); of a split block's pieces: the partial results before this one
};

// What the planning kernel leaves for the attention kernel.
struct PlanHead
{
	int n_pieces;
};

struct PromptWs
{
	int* err;
	PlanHead* head;
	int* blk0;       // [n_req + 1] blocks before request r
	int* tiles;      // [blocks] tiles of a block
	Piece* pieces;
	int* counters;   // [blocks][n_kv]
	float* parts;
	int* taken;      // [PLACES] whether a CTA has the place
	float* sums;     // [PLACES][D / 4][BR] of 4: what O held before it started anew
	int max_blocks, max_pieces;
};

// The tiles of rows [row0, row0 + n) of a request; lo > hi: no keys.
__device__ __forceinline__ void row_tiles(const Kv4Args& a, const Kv4Request& x, int rows, int row0, int n, int& lo, int& hi)
{
	lo = 1;
	hi = 0;
	if (row0 >= rows) return;
	const int p0 = x.pos0 + row0 / a.group, p1 = x.pos0 + (min(rows, row0 + n) - 1) / a.group;
	const int first = kv4_first_key(a, p0), last = min(p1, x.keys - 1);
	if (last < first) return;
	lo = first / BN;
	hi = last / BN;
}

__device__ __forceinline__ int prompt_rows(const Kv4Args& a, const Kv4Request& x, int min_rows)
{
	const int rows = x.n_new * a.group;
	return rows > min_rows ? rows : 0;
}

// Inclusive running sum over the CTA, and the total.
template <typename T>
__device__ __forceinline__ T plan_scan(T v, T* sums, T& total)
{
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1)
	{
		const T u = __shfl_up_sync(0xffffffffu, v, o);
		if (lane >= o) v += u;
	}
	__syncthreads();
	if (lane == 31) sums[warp] = v;
	__syncthreads();
	T before = 0, all = 0;
	for (int w = 0; w < PLAN_THREADS / 32; ++w)
	{
		if (w < warp) before += sums[w];
		all += sums[w];
	}
	total = all;
	return before + v;
}

template <int BR>
__global__ void __launch_bounds__(PLAN_THREADS) kv4_plan_kernel(const Kv4Args a, const PromptWs ws, int min_rows)
{
	__shared__ int sums[PLAN_THREADS / 32];
	__shared__ long long tile_sums[PLAN_THREADS / 32];
	const int tid = threadIdx.x;
	int at = 0, total;
	for (int r0 = 0; r0 < a.n_req; r0 += PLAN_THREADS)
	{
		const int r = r0 + tid;
		int nb = 0;
		if (r < a.n_req) nb = (prompt_rows(a, kv4_request(a, r), min_rows) + BR - 1) / BR;
		const int end = at + plan_scan(nb, sums, total);
		if (r < a.n_req) ws.blk0[r + 1] = min(end, ws.max_blocks);
		at += total;
	}
	if (tid == 0) ws.blk0[0] = 0;
	if (tid < PLACES) ws.taken[tid] = 0; // (a call that gave up may have left them)
	__syncthreads();
	const int blocks = min(at, ws.max_blocks);
	const auto find = [&](int b) {
		int lo = 0, hi = a.n_req - 1;
		while (lo < hi)
		{
			const int mid = (lo + hi + 1) >> 1;
			if (ws.blk0[mid] <= b)
				lo = mid;
			else
				hi = mid - 1;
		}
		return lo;
	};
	// the blocks' tiles, and what a piece may have of them
	long long mine = 0, tiles;
	for (int b = tid; b < blocks; b += PLAN_THREADS)
	{
		const int r = find(b);
		const Kv4Request x = kv4_request(a, r);
		int lo, hi;
		row_tiles(a, x, prompt_rows(a, x, min_rows), (b - ws.blk0[r]) * BR, BR, lo, hi);
		const int n = max(1, hi - lo + 1); // (a block without keys still writes its zeros)
		ws.tiles[b] = n;
		mine += n;
	}
	plan_scan(mine, tile_sums, tiles);
	const int longest = kv4_longest(tiles, a.n_kv);
	int pieces = 0, split = 0;
	for (int b0 = 0; b0 < blocks; b0 += PLAN_THREADS)
	{
		const int b = b0 + tid, n = b < blocks ? ws.tiles[b] : 0, np = n / longest + (n % longest > 0);
		int t1, t2;
		const int p1 = pieces + plan_scan(np, sums, t1), s1 = split + plan_scan(np > 1 ? np : 0, sums, t2);
		pieces += t1;
		split += t2;
		if (b < blocks)
		{
			const int r = find(b), row0 = (b - ws.blk0[r]) * BR;
			const Kv4Request x = kv4_request(a, r);
			int lo, hi;
			row_tiles(a, x, prompt_rows(a, x, min_rows), row0, BR, lo, hi);
			const int first = p1 - np, each = (n + np - 1) / np;
			for (int i = 0; i < np && first + i < ws.max_pieces; ++i)
				ws.pieces[first + i] = Piece{r, row0, (lo > hi ? 0 : lo) + i * each, min(each, n - i * each), first, np, b,
				                             s1 - np + i};
			for (int h = 0; h < a.n_kv; ++h) ws.counters[(size_t)b * a.n_kv + h] = 0;
		}
	}
	if (tid == 0) ws.head->n_pieces = min(pieces, ws.max_pieces);
}

// The products are issued by a whole warp, converged, and executed by its
// elected lane; every condition on their way is a vote, whose result the
// compiler knows to be one for the warp. The operands' descriptors then live
// in the warp's uniform registers. (From a branch that one lane takes, or
// under conditions that might differ between lanes, each product cost 80 to
// 260 cycles of moving them there, whatever its size.)
__device__ __forceinline__ bool uni(bool c) { return __any_sync(0xffffffffu, c) != 0; }
__device__ __forceinline__ uint32_t elect_one()
{
	uint32_t r;
	asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
	return r;
}
// D (+)= A B, both in shared memory: a, b the low words of their descriptors
// (address and leading offset), which share the high word.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t id, uint32_t acc,
                                       uint32_t lead)
{
	asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
	             "mov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %3};\n\t"
	             "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n\t}" ::"r"(d),
	             "r"(a), "r"(b), "r"(high), "r"(id), "r"(acc), "r"(lead)
	             : "memory");
}
// A in TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t id, uint32_t acc,
                                       uint32_t lead)
{
	asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
	             "mov.b64 y, {%2, %3};\n\t"
	             "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
	             "r"(a), "r"(b), "r"(high), "r"(id), "r"(acc), "r"(lead)
	             : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t lead)
{
	asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
	             "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
	             "r"(lead)
	             : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack_half2(float x, float y)
{
	const __half2 h = __floats2half2_rn(x, y);
	return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

template <int D>
__global__ void __launch_bounds__(PT, 1) kv4_prompt_kernel(const Kv4Args a, const PromptWs ws, int min_rows)
{
	using L = PShape<D>;
	constexpr int U = L::U, NQ = L::NQ, KS = L::KS, RS = L::RAW_STAGES;
	const int pid = (int)blockIdx.x / a.n_kv, hk = (int)blockIdx.x % a.n_kv;
	const int n_pieces = ws.head->n_pieces;
	if (pid >= n_pieces) return;
	const Piece pc = ws.pieces[n_pieces - 1 - pid]; // a request's last rows see the most keys: first
	extern __shared__ unsigned char smem_raw[];
	unsigned char* smem =
		reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
	uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::SM_BAR);
	uint64_t* raw_full = bars;          // [4] a half tile's codes and scales are here
	uint64_t* raw_empty = bars + 4;     // [4] the unpacking warps have read them
	uint64_t* k_full = bars + 8;        // [2] an unpacked K tile
	uint64_t* k_empty = bars + 10;      // [2] its products are done
	uint64_t* v_full = bars + 12;       // [2]
	uint64_t* v_empty = bars + 14;      // [2]
	uint64_t* s_full = bars + 16;       // [2 Q tiles][2 buffers]
	uint64_t* p_full = bars + 20;       // [2 Q tiles][2 buffers]: P in TMEM (and O rescaled)
	uint64_t* pv_done = bars + 24;      // [2] one phase per P V of the Q tile
	uint64_t* o_done = bars + 26;       // [2] its last P V is done
	uint64_t* q_ready = bars + 28;      // Q's halves are in shared memory
	uint64_t* mma_done = bars + 29;     // every product issued is done
	uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 30);
	volatile int* flags = reinterpret_cast<volatile int*>(bars + 31); // [0] abort, [1] a V scale was no number
	int* shared_last = reinterpret_cast<int*>(bars + 32);
	int* place = shared_last + 1; // where O's earlier sums go
	int* loaded = reinterpret_cast<int*>(bars + 33); // [16] by tile: which 16-key parts of it are in the cache
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

	const Kv4Request x = kv4_request(a, pc.r);
	const int rows = prompt_rows(a, x, min_rows);
	// each Q tile's key tiles within the piece; none: lo > hi
	int lo[2] = {1, 1}, hi[2] = {0, 0};
#pragma unroll
	for (int X = 0; X < NQ; ++X)
	{
		row_tiles(a, x, rows, pc.row0 + 128 * X, 128, lo[X], hi[X]);
		lo[X] = max(lo[X], pc.tile0);
		hi[X] = min(hi[X], pc.tile0 + pc.tiles - 1);
	}
	const bool any = lo[0] <= hi[0] || (NQ == 2 && lo[1] <= hi[1]);
	const int u_lo = pc.tile0, n_u = any ? pc.tiles : 0;

	if (threadIdx.x == 0)
	{
		for (int s = 0; s < 4; ++s)
		{
			mbar_init(&raw_full[s], 1);
			mbar_init(&raw_empty[s], 4);
			mbar_init(&s_full[s], 1);
			mbar_init(&p_full[s], 128);
		}
		for (int s = 0; s < 2; ++s)
		{
			mbar_init(&k_full[s], 128);
			mbar_init(&k_empty[s], 1);
			mbar_init(&v_full[s], 128);
			mbar_init(&v_empty[s], 1);
			mbar_init(&pv_done[s], 1);
			mbar_init(&o_done[s], 1);
		}
		mbar_init(q_ready, NQ * 128);
		mbar_init(mma_done, 1);
		flags[0] = flags[1] = 0;
		fence_barrier_init();
	}
	if (warp == 1) tmem_alloc(tmem_slot, L::COLS);
	if (threadIdx.x == 64)
	{
		// (The SM's number is where it looks first: no other CTA is likely to have that place. A try takes about 1 us. Kept
		// short: a longer form here, or one among the roles below, made the whole kernel 4 to 6 % slower.)
		uint32_t at;
		asm volatile("mov.u32 %0, %%smid;" : "=r"(at));
		at = at % PLACES;
		int was;
#pragma unroll 1
		for (int i = 0; (was = atomicCAS(ws.taken + at, 0, 1)) != 0 && i < PLACE_TRIES; ++i) at = at + 1 < PLACES ? at + 1 : 0;
		__threadfence();
		*place = was ? -1 : (int)at;
	}
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = *tmem_slot;
	if (*place < 0) flags[0] = 1, atomicCAS(ws.err, 0, DEVERR_PLAN);
	if (tmem != 0) flags[0] = 1, atomicCAS(ws.err, 0, DEVERR_PLAN); // (cannot be: see the products' warp)

	// registers to the softmax (the launch gives every thread 128: 128 x (72 + 104 + 2 x 168) = 512 x 128)
	if (warp < 4)
	{
		asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
		if (warp == 0)
		{
			// ---- codes and scales: lane = 2 x part of the tile + {codes, scales} ----
			const int parts = min(BN, a.page), n_parts = BN / parts;
			const int what = lane & 1, part = lane >> 1;
			const int row_bytes = what ? U * 2 : D / 2;
			const int cb = kv4_codes_bytes(a.page, D), sb = kv4_scales_bytes(a.page, D);
			const int* table = a.table + (size_t)pc.r * a.table_stride;
			const int last = min(x.pos0 + x.n_new - 1, x.keys - 1);
			int ids = -1, base = -1, h = 0;
			int id[2] = {-1, -1}; // this lane's page of the K tile and of the V tile behind it
			unsigned got[2] = {0, 0};
			const auto load = [&](int v, int u) {
				const int s = h % RS;
				if (h >= RS && !flags[0] && !kv4_wait(&raw_empty[s], ((h / RS) - 1) & 1, ws.err, DEVERR_WAIT_EMPTY))
					flags[0] = 1;
				__syncwarp();
				if (__shfl_sync(0xffffffffu, flags[0], 0)) return false;
				const int k0 = (u_lo + u) * BN + part * parts;
				if (lane == 0) mbar_arrive_expect_tx(&raw_full[s], __popc(got[v]) / 2 * (uint32_t)(parts * (D / 2 + U * 2)));
				__syncwarp();
				if (got[v] >> lane & 1)
				{
					const int off = k0 & (a.page - 1);
					bulk_g2s(smem + L::SM_RAW + s * L::RAW + (what ? L::CODES : 0) + part * parts * row_bytes,
					         a.pages + ((size_t)id[v] * a.n_kv + hk) * kv4_chunk_bytes(a.page, D) +
					             (what ? 2 * cb + v * sb : v * cb) + off * row_bytes,
					         parts * row_bytes, &raw_full[s]);
				}
				++h;
				return true;
			};
			bool ok = true;
			for (int u = 0; ok && u <= n_u; ++u)
			{
				if (u > 0) id[1] = id[0], got[1] = got[0];
				if (u < n_u)
				{
					const int page0 = ((u_lo + u) * BN) >> a.page_shift;
					if (base < 0 || page0 + n_parts > base + 32)
					{
						base = page0;
						ids = base + lane < a.max_blocks ? table[base + lane] : -1;
					}
					id[0] = __shfl_sync(0xffffffffu, ids, page0 - base + (part < n_parts ? part : 0));
					const bool get = part < n_parts && id[0] >= 0 && id[0] < a.n_pages && (u_lo + u) * BN + part * parts <= last;
					got[0] = __ballot_sync(0xffffffffu, get);
					if (lane == 0)
					{
						int mask = 0;
						for (int p = 0; p < n_parts; ++p)
							if (got[0] >> (2 * p) & 1) mask |= ((1 << (parts / 16)) - 1) << (p * (parts / 16));
						loaded[u & 15] = mask;
					}
					ok = load(0, u);
				}
				if (ok && u > 0) ok = load(1, u - 1);
			}
			// not to leave (after a wait that ran out) while a copy may still land here
			for (int i = max(0, h - RS); i < h; ++i) kv4_wait(&raw_full[i % RS], (i / RS) & 1, nullptr, 0);
			__syncwarp();
		}
		else if (warp == 1)
		{
			constexpr uint32_t ID_S = tc_idesc(128, BN, false, false, false);
			constexpr uint32_t ID_PV = tc_idesc(128, D, false, false, true);
			const uint32_t lead = elect_one();
			constexpr uint32_t tm = 0; // (512 columns are all there are: the allocation starts at the first)
			const uint32_t dq = (uint32_t)sdesc(smem_u32(smem + L::SM_Q), 16, 1024);
			const uint32_t dk = (uint32_t)sdesc(smem_u32(smem + L::SM_K), 16, 1024);
			const uint32_t dv = (uint32_t)sdesc(smem_u32(smem + L::SM_V), L::KV_PANEL, 1024);
			const uint32_t high = (uint32_t)(sdesc(0, 16, 1024) >> 32);
			const auto has = [&](int X, int u) { return uni(u + u_lo >= lo[X] && u + u_lo <= hi[X]); };
			int ns[2] = {0, 0}, np[2] = {0, 0}; // S issued, P consumed, per Q tile
			const auto wait = [&](uint64_t* bar, int phase) {
				const bool w = !flags[0] && kv4_wait(bar, (uint32_t)(phase & 1), ws.err, DEVERR_WAIT_FULL);
				return __all_sync(0xffffffffu, w) != 0;
			};
			// (the low halves first: the adder cuts a sum off at its size, and while only they are in it that is small)
			const auto issue_s = [&](int X, int u) {
				const bool odd = uni(ns[X] & 1);
				const uint32_t d = tm + 128 * X + (odd ? 64 : 0);
				const uint32_t q = dq + 2 * X * (L::Q_HALF >> 4), k = dk + (u % KS) * (L::KV_TILE >> 4);
#pragma unroll
				for (int half = 1; half >= 0; --half)
#pragma unroll
					for (int i = 0; i < D / 16; ++i)
						mma_ss(d, q + half * (L::Q_HALF >> 4) + (i >> 2) * (L::Q_PANEL >> 4) + (i & 3) * 2,
						       k + (i >> 2) * (L::KV_PANEL >> 4) + (i & 3) * 2, high, ID_S, half == 0 || i > 0, lead);
				commit(&s_full[2 * X + odd], lead);
				++ns[X];
			};
			bool ok = uni(n_u == 0) || wait(q_ready, 0);
			for (int u = 0; u < 2 && uni(ok && u < n_u); ++u)
			{
				ok = wait(&k_full[u % KS], u / KS);
				if (!ok) break;
				tc_fence_after();
#pragma unroll
				for (int X = 0; X < NQ; ++X)
					if (has(X, u)) issue_s(X, u);
				commit(&k_empty[u % KS], lead);
			}
			for (int u = 0; uni(ok && u < n_u); ++u)
			{
				const int s = u % KS;
				ok = wait(&v_full[s], u / KS);
				const bool ahead = uni(u + 2 < n_u);
				bool k_ready = false;
#pragma unroll
				for (int X = 0; X < NQ; ++X)
				{
					if (ok && has(X, u))
					{
						const bool odd = uni(np[X] & 1);
						ok = wait(&p_full[2 * X + odd], np[X] >> 1);
						if (ok)
						{
							tc_fence_after();
							const uint32_t d = tm + L::T_O + D * X, p = tm + 128 * X + (odd ? 64 : 0);
							const uint32_t v = dv + s * (L::KV_TILE >> 4);
							const bool more = uni(np[X] % FRESH > 0);
#pragma unroll
							for (int i = 0; i < BN / 16; ++i)
							{
								mma_ts(d, p + 8 * i, v + 128 * i, high, ID_PV, i > 0 ? 1 : more, lead);
								mma_ts(d, p + 32 + 8 * i, v + 128 * i, high, ID_PV, 1, lead);
							}
							commit(&pv_done[X], lead);
							if (uni(u + u_lo == hi[X])) commit(&o_done[X], lead);
							++np[X];
						}
					}
					if (X == NQ - 1) commit(&v_empty[s], lead);
					if (ok && ahead && has(X, u + 2))
					{
						if (!k_ready)
						{
							ok = wait(&k_full[(u + 2) % KS], (u + 2) / KS);
							tc_fence_after();
							k_ready = true;
						}
						if (ok) issue_s(X, u + 2);
					}
				}
				if (ok && ahead)
				{
					if (!k_ready) ok = wait(&k_full[(u + 2) % KS], (u + 2) / KS);
					commit(&k_empty[(u + 2) % KS], lead);
				}
			}
			if (!ok) flags[0] = 1;
			commit(mma_done, lead);
			kv4_wait(mma_done, 0, nullptr, 0);
			__syncwarp();
		}
	}
	else if (warp < 8)
	{
		asm volatile("setmaxnreg.dec.sync.aligned.u32 104;" ::: "memory");
		// ---- unpacking: a thread takes words (8 codes) of a half tile ----
		const int tid = threadIdx.x - 128;
		constexpr int WPR = D / 8, WORDS = BN * WPR / 128; // words a row; a thread's of a half tile
		int h = 0;
		const auto unpack = [&](auto which, int u) {
			constexpr bool V = decltype(which)::value;
			constexpr int v = V;
			const int rs = h % RS, s = u % KS;
			uint64_t* empty = v ? v_empty : k_empty;
			bool ok = !flags[0] && kv4_wait(&raw_full[rs], (h / RS) & 1, ws.err, DEVERR_WAIT_FULL);
			ok = ok && (u < KS || (!flags[0] && kv4_wait(&empty[s], ((u / KS) - 1) & 1, ws.err, DEVERR_WAIT_EMPTY)));
			if (!__all_sync(0xffffffffu, ok))
			{
				flags[0] = 1;
				return false;
			}
			const unsigned char* raw = smem + L::SM_RAW + rs * L::RAW;
			unsigned char* dst = smem + (v ? L::SM_V : L::SM_K) + s * L::KV_TILE;
			const int key0 = (u_lo + u) * BN;
			bool odd = false;
			constexpr int BATCH = WORDS < 8 ? WORDS : 8; // read before any is written: the stores could be to their place
#pragma unroll
			for (int i0 = 0; i0 < WORDS; i0 += BATCH)
			{
				uint32_t c[BATCH];
				float f[BATCH];
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
				{
					const int at = tid + 128 * (i0 + i), row = at / WPR, g = kv4_unit(row, at % WPR >> 2, D);
					c[i] = *reinterpret_cast<const uint32_t*>(raw + 4 * at);
					f[i] = bf16_bits_to_float(*reinterpret_cast<const uint16_t*>(raw + L::CODES + (row * U + g) * 2));
				}
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
				{
					const int at = tid + 128 * (i0 + i), row = at / WPR, w = at % WPR;
					const int chunk = 4 * kv4_unit(row, w >> 2, D) + (w & 3); // 8 values: 16 bytes unpacked
					if constexpr (V)
					{
						// no number (or whatever lies past the keys): zero weights must stay zero. Rows that see such a
						// key of theirs get none at the end.
						const bool fine = fabsf(f[i]) <= KV4_SCALE_MAX;
						odd |= !fine && key0 + row < x.keys;
						f[i] = fine ? f[i] : 0.0f;
					}
					const __half2 sc = __float2half2_rn(f[i]);
					uint32_t y[4];
#pragma unroll
					for (int e = 0; e < 4; ++e)
					{
						const uint32_t z = e >= 2 ? c[i] >> 8 : c[i];
						uint32_t m = e & 1 ? (z & 0x00F000F0u) | 0x54005400u : (z & 0x000F000Fu) | 0x64006400u;
						const __half2 q =
							__hmul2(__hadd2(*reinterpret_cast<__half2*>(&m), __float2half2_rn(e & 1 ? -72.0f : -1032.0f)), sc);
						y[e] = *reinterpret_cast<const uint32_t*>(&q);
					}
					*reinterpret_cast<uint4*>(dst + (chunk >> 3) * L::KV_PANEL + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) =
						make_uint4(y[0], y[1], y[2], y[3]);
				}
			}
			if (odd) flags[1] = 1;
			fence_async_shared();
			mbar_arrive(v ? &v_full[s] : &k_full[s]);
			__syncwarp();
			if (lane == 0) mbar_arrive(&raw_empty[rs]);
			++h;
			return true;
		};
		bool ok = true;
		for (int u = 0; ok && u <= n_u; ++u)
		{
			if (u < n_u) ok = unpack(std::false_type{}, u);
			if (ok && u > 0) ok = unpack(std::true_type{}, u - 1);
		}
	}
	else
	{
		asm volatile("setmaxnreg.inc.sync.aligned.u32 168;" ::: "memory");
		const int X = (warp - 8) >> 2, wq = warp & 3, r = wq * 32 + lane;
		if (X < NQ)
		{
			const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
			const uint32_t ts0 = tmem + 128 * X + lane_off, to = tmem + L::T_O + D * X + lane_off;
			const int row = pc.row0 + 128 * X + r, tok = row / a.group;
			const bool real = row < rows;
			const int qp = x.pos0 + tok;
			const int kf = kv4_first_key(a, qp), kl = real ? min(qp, x.keys - 1) : -1;

			// ---- the warp's 32 rows of Q, as two 16-bit halves: whole rows, LPR lanes each ----
			constexpr int LPR = D / 4 < 32 ? D / 4 : 32, VPL = D / 4 / LPR, RPI = 32 / LPR;
			constexpr int BATCH = 8 / VPL; // row loads in flight
			unsigned char* qs = smem + L::SM_Q + X * 2 * L::Q_HALF;
			float f = 1.0f; // this thread's row's factor
#pragma unroll 1
			for (int i0 = 0; i0 < 32; i0 += RPI * BATCH)
			{
				float4 y[BATCH][VPL];
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
				{
					const int rw = pc.row0 + 128 * X + wq * 32 + i0 + i * RPI + lane / LPR, tk = rw / a.group;
					const float* q = a.q + (size_t)(x.q0 + tk) * a.q_stride + (size_t)(hk * a.group + rw - tk * a.group) * D;
#pragma unroll
					for (int j = 0; j < VPL; ++j)
						y[i][j] = rw < rows ? *reinterpret_cast<const float4*>(q + 4 * (lane % LPR + j * LPR))
						                    : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				}
				float tops[BATCH];
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
				{
					tops[i] = 0.0f;
#pragma unroll
					for (int j = 0; j < VPL; ++j)
						tops[i] = fmaxf(tops[i], fmaxf(fmaxf(fabsf(y[i][j].x), fabsf(y[i][j].y)), fmaxf(fabsf(y[i][j].z), fabsf(y[i][j].w))));
				}
#pragma unroll
				for (int o = LPR / 2; o > 0; o >>= 1)
#pragma unroll
					for (int i = 0; i < BATCH; ++i) tops[i] = fmaxf(tops[i], __shfl_xor_sync(0xffffffffu, tops[i], o));
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
				{
					const float top = tops[i];
					const int ex = top > 0.0f ? max(-100, min(100, ilogbf(top))) : 0;
					// the largest to [2^13, 2^14); the scale's sign too, so that mult below has none
					const float g = copysignf(__uint_as_float((uint32_t)(127 + 13 - ex) << 23), a.scale);
					const int first = i0 + i * RPI, rr = wq * 32 + first + lane / LPR;
					const float g2 = __shfl_sync(0xffffffffu, g, (lane - first) * LPR & 31);
					if (lane >= first && lane < first + RPI) f = g2;
#pragma unroll
					for (int j = 0; j < VPL; ++j)
					{
						const float4 z = make_float4(y[i][j].x * g, y[i][j].y * g, y[i][j].z * g, y[i][j].w * g);
						const uint32_t h0 = pack_half2(z.x, z.y), h1 = pack_half2(z.z, z.w);
						const float2 b0 = unpack_half2(h0), b1 = unpack_half2(h1);
						const int c = (lane % LPR + j * LPR) >> 1; // the 16-byte chunk: this lane has one half of it
						unsigned char* dst = qs + (c >> 3) * L::Q_PANEL + rr * 128 + (((c & 7) ^ (rr & 7)) << 4) + (lane & 1) * 8;
						*reinterpret_cast<uint2*>(dst) = make_uint2(h0, h1);
						*reinterpret_cast<uint2*>(dst + L::Q_HALF) = make_uint2(pack_half2(z.x - b0.x, z.y - b0.y), pack_half2(z.z - b1.x, z.w - b1.y));
					}
				}
			}
			fence_async_shared();
			mbar_arrive(q_ready);

			// ---- the softmax, O kept in scale ----
			// (never zero: a masked score times mult stays -infinity. The least normal float leaves any score at zero.)
			const float mult = fmaxf((a.softcap > 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f) / f, FLT_MIN);
			const float cap2 = a.softcap * 1.4426950408889634f;
			// HELD - held score (1e30: no key seen; places without a row: any score, for they never see one)
			float held = real ? 1e30f : 0.0f, l = 0.0f;
			// O's earlier parts, relative to sums_held
			float4* sums = reinterpret_cast<float4*>(ws.sums + (size_t)max(*place, 0) * L::BR * D) + 128 * X + r;
			float sums_held = 0.0f;
			bool have_sums = false;
			const auto add_up = [&](float now) {
				const float by = have_sums ? ex2(now - sums_held) : 0.0f;
#pragma unroll
				for (int c = 0; c < D; c += 32)
				{
					float o[32];
					tmem_ld32(to + c, o);
					float4 y[8];
#pragma unroll
					for (int i = 0; i < 8; ++i)
						y[i] = have_sums ? __ldcg(sums + (c / 4 + i) * L::BR) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
					tmem_wait_ld();
#pragma unroll
					for (int i = 0; i < 8; ++i)
						__stcg(sums + (c / 4 + i) * L::BR,
						       make_float4(fmaf(y[i].x, by, o[4 * i]), fmaf(y[i].y, by, o[4 * i + 1]), fmaf(y[i].z, by, o[4 * i + 2]),
						                   fmaf(y[i].w, by, o[4 * i + 3])));
				}
				have_sums = true;
			};
			bool ok = true;
			int n = 0;
			const int t_lo = X ? lo[1] : lo[0], t_hi = X ? hi[1] : hi[0];
			for (int t = t_lo; t <= t_hi; ++t, ++n)
			{
				const int b = n & 1;
				const uint32_t ts = ts0 + 64 * b;
				ok = ok && !flags[0] && kv4_wait(&s_full[2 * X + b], (uint32_t)((n >> 1) & 1), ws.err, DEVERR_WAIT_FULL);
				if (!__all_sync(0xffffffffu, ok))
				{
					ok = false;
					break;
				}
				tc_fence_after();
				float s[BN];
				tmem_ld32(ts, s);
				tmem_ld32(ts + 32, s + 32);
				tmem_wait_ld();
				if (a.softcap > 0.0f)
				{
#pragma unroll
					for (int c = 0; c < BN; ++c) s[c] = tanhf(s[c] * mult) * cap2;
				}
				const float sl = a.softcap > 0.0f ? 1.0f : mult;
				const int key0 = t * BN, here = loaded[(t - u_lo) & 15];
				if (key0 < kf || key0 + BN - 1 > kl || here != 15)
				{
#pragma unroll
					for (int c = 0; c < BN; ++c)
						if (key0 + c < kf || key0 + c > kl || !(here >> (c >> 4) & 1)) s[c] = -CUDART_INF_F;
				}
				// weights against the held score; `over`: the largest exponent
				float sum[4];
				const auto write_p = [&](float h) {
					float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
					for (int i = 0; i < 4; ++i) sum[i] = 0.0f;
#pragma unroll
					for (int c0 = 0; c0 < BN; c0 += 32)
					{
						float ph[16], pl[16]; // pairs of 16-bit halves
#pragma unroll
						for (int c = c0; c < c0 + 32; c += 2)
						{
							const float e0 = fmaf(s[c], sl, h), e1 = fmaf(s[c + 1], sl, h);
							mx[(c >> 1) & 3] = fmaxf(mx[(c >> 1) & 3], fmaxf(e0, e1));
							const float p0 = ex2(e0), p1 = ex2(e1);
							sum[(c >> 1) & 3] += p0 + p1;
							const uint32_t w = pack_half2(p0, p1);
							const float2 y = unpack_half2(w);
							ph[(c - c0) >> 1] = __uint_as_float(w);
							pl[(c - c0) >> 1] = __uint_as_float(pack_half2(p0 - y.x, p1 - y.y));
						}
						tmem_st<16>(ts + c0 / 2, ph);
						tmem_st<16>(ts + 32 + c0 / 2, pl);
					}
					return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
				};
				const float before = held; // what O is relative to
				float alpha = 1.0f;
				bool move;
				if (__any_sync(0xffffffffu, held == 1e30f))
				{
					// a row's first keys: the tile's maximum first
					float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
					for (int c = 0; c < BN; ++c) mx[c & 3] = fmaxf(mx[c & 3], s[c] * sl);
					const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
					move = m + held > HELD_TOP;
					if (move)
					{
						alpha = ex2(HELD - m - held); // (none seen before: 0)
						held = HELD - m;
					}
					write_p(held);
				}
				else
				{
					const float over = write_p(held);
					move = over > HELD_TOP;
					if (__any_sync(0xffffffffu, move))
					{
						if (move)
						{
							alpha = ex2(HELD - over);
							held += HELD - over;
						}
						tmem_wait_st(); // (stores that are under way need not land in their order)
						write_p(held);
					}
				}
				const bool fresh = n > 0 && n % FRESH == 0;
				if (fresh || (__any_sync(0xffffffffu, move) && n > 0))
				{
					// O must hold every P V before this tile's. (S of this tile completed after P V of tile n - 2, so
					// pv_done is at most one phase behind and its parity does not alias.)
					const bool done = !flags[0] && kv4_wait(&pv_done[X], (uint32_t)((n - 1) & 1), ws.err, DEVERR_WAIT_FULL);
					if (!__all_sync(0xffffffffu, done))
					{
						ok = false;
						break;
					}
					tc_fence_after();
					if (fresh)
					{
						add_up(before);
						sums_held = before;
					}
					else
#pragma unroll
						for (int c = 0; c < D; c += 32)
						{
							float o[32];
							tmem_ld32(to + c, o);
							tmem_wait_ld();
#pragma unroll
							for (int i = 0; i < 32; ++i) o[i] *= alpha;
							tmem_st32(to + c, o);
						}
				}
				tmem_wait_st();
				l = fmaf(l, alpha, (sum[0] + sum[1]) + (sum[2] + sum[3]));
				tc_fence_before();
				mbar_arrive(&p_full[2 * X + b]);
			}
			if (!ok) flags[0] = 1;
			if (ok && n > 0) ok = !flags[0] && kv4_wait(&o_done[X], 0, ws.err, DEVERR_WAIT_FULL);
			ok = __all_sync(0xffffffffu, ok);
			tc_fence_after();

			// ---- the row's output, or its part of it ----
			const bool spoilt = flags[1] != 0;
			const float inv = l == 0.0f ? 0.0f : 1.0f / l;
			// (this Q tile is not read any more, nor, after the barrier, still being written: O goes out through its
			// place, whole rows at a time)
			named_sync(2 + X, 128);
			unsigned char* os = smem + L::SM_Q + X * 2 * L::Q_HALF + wq * 32 * (D * 4);
			const auto stage_out = [&](int c, const float (&o)[32], float by) {
#pragma unroll
				for (int i = 0; i < 32; i += 4)
					*reinterpret_cast<float4*>(os + lane * (D * 4) + ((((c + i) / 4) ^ (lane & 7)) << 4)) =
						make_float4(o[i] * by, o[i + 1] * by, o[i + 2] * by, o[i + 3] * by);
			};
			const auto rows_out = [&]() {
				__syncwarp();
#pragma unroll 4
				for (int i = 0; i < 32; i += RPI)
				{
					const int in = i + lane / LPR, rw = pc.row0 + 128 * X + wq * 32 + in, tk = rw / a.group;
					if (rw >= rows) continue;
					float* dst = a.out + (size_t)(x.q0 + tk) * a.out_stride + (size_t)(hk * a.group + rw - tk * a.group) * D;
#pragma unroll
					for (int j = 0; j < VPL; ++j)
					{
						const int c = lane % LPR + j * LPR;
						*reinterpret_cast<float4*>(dst + 4 * c) =
							*reinterpret_cast<const float4*>(os + in * (D * 4) + ((c ^ (in & 7)) << 4));
					}
				}
			};
			const auto slot = [&](int i) { // piece i of the block
				return ws.parts + ((size_t)(pc.split0 - (n_pieces - 1 - pid - pc.first) + i) * a.n_kv + hk) * L::PART;
			};
			const int my = n_pieces - 1 - pid - pc.first;
#pragma unroll 1
			for (int c = 0; c < D; c += 32)
			{
				float o[32];
				if (n > 0)
				{
					tmem_ld32(to + c, o);
					tmem_wait_ld();
				}
				else
#pragma unroll
					for (int i = 0; i < 32; ++i) o[i] = 0.0f;
				if (have_sums)
				{
					const float by = ex2(held - sums_held);
#pragma unroll
					for (int i = 0; i < 8; ++i)
					{
						const float4 y = __ldcg(sums + (c / 4 + i) * L::BR);
						o[4 * i] = fmaf(y.x, by, o[4 * i]), o[4 * i + 1] = fmaf(y.y, by, o[4 * i + 1]);
						o[4 * i + 2] = fmaf(y.z, by, o[4 * i + 2]), o[4 * i + 3] = fmaf(y.w, by, o[4 * i + 3]);
					}
				}
				if (spoilt && real)
				{
					// (32 columns are one group of values)
					const int from = max(kf, pc.tile0 * BN), to_ = min(kl, (pc.tile0 + pc.tiles) * BN - 1);
					for (int k = from; k <= to_; ++k)
					{
						const int id = a.table[(size_t)pc.r * a.table_stride + (k >> a.page_shift)];
						if (id < 0 || id >= a.n_pages) continue;
						const uint8_t* chunk = a.pages + ((size_t)id * a.n_kv + hk) * kv4_chunk_bytes(a.page, D);
						const uint16_t* vs = reinterpret_cast<const uint16_t*>(chunk + 2 * kv4_codes_bytes(a.page, D) +
						                                                       kv4_scales_bytes(a.page, D));
						const float f2 = bf16_bits_to_float(vs[(k & (a.page - 1)) * U + c / KV4_GROUP]);
						if (!(fabsf(f2) <= KV4_SCALE_MAX))
#pragma unroll
							for (int i = 0; i < 32; ++i) o[i] = CUDART_NAN_F;
					}
				}
				if (pc.n == 1)
					stage_out(c, o, inv);
				else
				{
					float4* p = reinterpret_cast<float4*>(slot(my)) + (c / 4) * L::BR + 128 * X + r;
#pragma unroll
					for (int i = 0; i < 32; i += 4) p[(i / 4) * L::BR] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
				}
			}
			if (pc.n == 1)
				rows_out();
			else
			{
				reinterpret_cast<float2*>(slot(my) + (size_t)L::BR * D)[128 * X + r] =
					make_float2(held == 1e30f ? -CUDART_INF_F : HELD - held, l);
				__threadfence();
				named_sync(1, NQ * 128);
				if (threadIdx.x == 256) *shared_last = atomicAdd(&ws.counters[(size_t)pc.block * a.n_kv + hk], 1) == pc.n - 1;
				named_sync(1, NQ * 128);
				if (*shared_last)
				{
					__threadfence();
					float m = -CUDART_INF_F, w = 0.0f;
					for (int i = 0; i < pc.n; ++i)
						m = fmaxf(m, __ldcg(reinterpret_cast<const float2*>(slot(i) + (size_t)L::BR * D) + 128 * X + r).x);
					for (int i = 0; i < pc.n; ++i)
					{
						const float2 z = __ldcg(reinterpret_cast<const float2*>(slot(i) + (size_t)L::BR * D) + 128 * X + r);
						w = fmaf(z.y, z.x == m ? 1.0f : ex2(z.x - m), w);
					}
					const float winv = w == 0.0f ? 0.0f : 1.0f / w;
#pragma unroll 1
					for (int c = 0; c < D; c += 32)
					{
						float o[32];
#pragma unroll
						for (int e = 0; e < 32; ++e) o[e] = 0.0f;
						for (int i = 0; i < pc.n; ++i)
						{
							const float zx = __ldcg(reinterpret_cast<const float2*>(slot(i) + (size_t)L::BR * D) + 128 * X + r).x;
							const float g = zx == m ? 1.0f : ex2(zx - m);
							const float4* p = reinterpret_cast<const float4*>(slot(i)) + (c / 4) * L::BR + 128 * X + r;
#pragma unroll
							for (int e = 0; e < 8; ++e)
							{
								const float4 y = __ldcg(p + e * L::BR);
								o[4 * e] = fmaf(y.x, g, o[4 * e]), o[4 * e + 1] = fmaf(y.y, g, o[4 * e + 1]);
								o[4 * e + 2] = fmaf(y.z, g, o[4 * e + 2]), o[4 * e + 3] = fmaf(y.w, g, o[4 * e + 3]);
							}
						}
						stage_out(c, o, winv);
					}
					rows_out();
				}
			}
		}
	}
	tc_fence_before();
	__syncthreads();
	if (threadIdx.x == 64 && *place >= 0)
	{
		__threadfence();
		atomicExch(ws.taken + *place, 0); // (the barrier has gathered every use of it)
	}
	if (warp == 1)
	{
		tc_fence_after();
		tmem_dealloc(tmem, L::COLS);
	}
}

size_t up(size_t x) { return (x + 255) / 256 * 256; }

// The workspace's parts behind `base` (which may be NULL: sizes only).
template <int D>
size_t prompt_ws(unsigned char* base, size_t at, int n_req, long long rows, int n_kv, PromptWs& ws)
{
	using L = PShape<D>;
	// every block but a request's last is full; a block cut into n pieces holds more than n - 1 shares
	const long long blocks = rows / L::BR + n_req, pieces = blocks + KV4_SHARES;
	ws.max_blocks = (int)blocks;
	ws.max_pieces = (int)pieces;
	const auto take = [&](size_t bytes) {
		unsigned char* p = base + at;
		at += up(bytes);
		return p;
	};
	ws.err = reinterpret_cast<int*>(base);
	ws.head = reinterpret_cast<PlanHead*>(take(sizeof(PlanHead)));
	ws.blk0 = reinterpret_cast<int*>(take(4 * ((size_t)n_req + 1)));
	ws.tiles = reinterpret_cast<int*>(take(4 * (size_t)blocks));
	ws.pieces = reinterpret_cast<Piece*>(take(sizeof(Piece) * (size_t)pieces));
	ws.counters = reinterpret_cast<int*>(take(4 * (size_t)blocks * n_kv));
	ws.parts = reinterpret_cast<float*>(take((size_t)2 * KV4_SHARES * L::PART * 4));
	ws.taken = reinterpret_cast<int*>(take(PLACES * 4));
	ws.sums = reinterpret_cast<float*>(take((size_t)PLACES * L::BR * D * 4));
	return at;
}

template <int D>
int launch(const Kv4Args& a, unsigned char* workspace, size_t at, int min_rows, cudaStream_t st)
{
	using L = PShape<D>;
	static bool configured[64] = {};
	int dev = 0;
	cudaGetDevice(&dev);
	if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
	auto kernel = kv4_prompt_kernel<D>;
	if (!configured[dev])
	{
		const cudaError_t ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
		if (ce != cudaSuccess) return (int)ce;
		configured[dev] = true;
	}
	PromptWs ws;
	prompt_ws<D>(workspace, at, a.n_req, (long long)a.n_tok * a.group, a.n_kv, ws);
	kv4_plan_kernel<L::BR><<<1, PLAN_THREADS, 0, st>>>(a, ws, min_rows);
	kernel<<<(unsigned)ws.max_pieces * (unsigned)a.n_kv, PT, L::SMEM, st>>>(a, ws, min_rows);
	note_launches(2);
	return (int)cudaGetLastError();
}

} // namespace

size_t kv4_prompt_ws_end(int D, size_t at, int n_req, long long rows, int n_kv)
{
	PromptWs ws;
	return D == 64    ? prompt_ws<64>(nullptr, at, n_req, rows, n_kv, ws)
	       : D == 128 ? prompt_ws<128>(nullptr, at, n_req, rows, n_kv, ws)
	                  : prompt_ws<256>(nullptr, at, n_req, rows, n_kv, ws);
}

int launch_kv4_prompt(const Kv4Args& a, void* workspace, size_t at, int min_rows, void* stream)
{
	unsigned char* w = static_cast<unsigned char*>(workspace);
	const auto st = static_cast<cudaStream_t>(stream);
	return a.D == 64    ? launch<64>(a, w, at, min_rows, st)
	       : a.D == 128 ? launch<128>(a, w, at, min_rows, st)
	                    : launch<256>(a, w, at, min_rows, st);
}

} // namespace nncu
