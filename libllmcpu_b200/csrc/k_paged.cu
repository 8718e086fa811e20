// k_paged.cu -- the paged cache's small operators: a step's tables from the
// requests' lengths, the rotation by per-token positions with several axes,
// and the 4-bit cache's write and read-back. (The attention over it:
// k_kv4_attn.cu.)
#include <cuda_runtime.h>

#include <cstdio>

#include "kv4.cuh"

namespace nncu
{
namespace
{

// ---- a step's tables ---------------------------------------------------------------
//
// Everything follows from three running sums over the requests: of their new
// tokens, of the pages they lack and of the pages they give back. Every CTA
// forms all three (12 bytes a request from L2, a scan in shared memory)
// instead of waiting for another one, then handles its share of the tokens,
// the new pages and the returned pages: one launch, no workspace. Bound by the
// launch and its dependent loads: 256 requests 5.8 us, 60 requests with 65 K
// tokens 7.6 us.

constexpr int STEP_THREADS = 512, STEP_WARPS = STEP_THREADS / 32;
// Running sums of absurd lengths stop here instead of wrapping: the sum of two such ends still fits an int. What goes
// into a sum is held to it too. The bit above says that the request is served.
constexpr int SAT = (1 << 30) - 1, SERVED = 1 << 30;

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, SAT); }

// Inclusive running sum over the CTA's threads; `total` gets the sum of all.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total)
{
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1)
	{
		const int u = __shfl_up_sync(0xffffffffu, v, o);
		if (lane >= o) v = sat_add(v, u);
	}
	__syncthreads(); // the previous call's sums have been read
	if (lane == 31) warp_sums[warp] = v;
	__syncthreads();
	int before = 0, all = 0;
#pragma unroll
	for (int w = 0; w < STEP_WARPS; ++w)
	{
		const int s = warp_sums[w];
		if (w < warp) before = sat_add(before, s);
		all = sat_add(all, s);
	}
	total = all;
	return sat_add(before, v);
}

// The last i of [0, n] with a[i] <= x (a rising, a[0] <= x), in the bits of MASK.
template <int MASK = -1>
__device__ __forceinline__ int last_at_most(const int* a, int n, int x)
{
	int lo = 0, hi = n;
	while (lo < hi)
	{
		const int mid = (lo + hi + 1) >> 1;
		if ((a[mid] & MASK) <= x)
			lo = mid;
		else
			hi = mid - 1;
	}
	return lo;
}

__global__ void __launch_bounds__(STEP_THREADS) paged_step_kernel(const nncu_paged_step s)
{
	extern __shared__ int sm[];
	const int n = s.n_req;
	int* tok = sm;             // [n + 1] running sum of new tokens
	int* lack = sm + (n + 1);  // [n + 1] ... of pages to take
	int* back = lack + n + 1;  // [n + 1] ... of pages given back, and whether the request before is SERVED
	__shared__ int warp_sums[STEP_WARPS];
	const long long room = (long long)s.max_blocks * s.page_size;
	const int np = s.n_pages, count = max(0, min(s.queue[1], np));

	if (threadIdx.x == 0) tok[0] = lack[0] = back[0] = 0;
	int c_tok = 0, c_lack = 0, c_back = 0;
	for (int i0 = 0; i0 < n; i0 += STEP_THREADS)
	{
		const int i = i0 + (int)threadIdx.x;
		int nn = 0, past = 0, held = 0, t;
		if (i < n)
		{
			nn = s.n_new[i];
			past = s.past[i];
			held = max(0, min(s.held[i], s.max_blocks));
		}
		const bool ends = nn < 0;
		const int q_end = sat_add(c_tok, block_scan(min(max(nn, 0), SAT), warp_sums, t));
		c_tok = sat_add(c_tok, t);
		const bool fits = !ends && past >= 0 && (long long)past + nn <= room && q_end <= s.max_tok;
		const int need = fits ? max(0, (int)(((long long)past + nn + s.page_size - 1) / s.page_size) - held) : 0;
		const int l_end = sat_add(c_lack, block_scan(min(need, SAT), warp_sums, t));
		c_lack = sat_add(c_lack, t);
		const int b_end = sat_add(c_back, block_scan(ends ? min(held, SAT) : 0, warp_sums, t));
		c_back = sat_add(c_back, t);
		// (Behind a request that the ring did not suffice for, one that lacks no page is served still.)
		const bool ok = fits && (need == 0 || l_end <= count);
		if (i < n) tok[i + 1] = q_end, lack[i + 1] = l_end, back[i + 1] = b_end | (ok ? SERVED : 0);
	}
	__syncthreads();

	const int head = ((s.queue[0] % np) + np) % np;
	const int taken = lack[last_at_most(lack, n, count)], given = back[n] & SAT;
	const int step = gridDim.x * STEP_THREADS, me = blockIdx.x * STEP_THREADS + (int)threadIdx.x;

	for (int r = me; r < n; r += step)
	{
		const int nn = s.n_new[r], past = s.past[r], held = max(0, min(s.held[r], s.max_blocks));
		const bool ok = back[r + 1] & SERVED;
		s.held_out[r] = nn < 0 ? 0 : held + (ok ? lack[r + 1] - lack[r] : 0);
		s.seq_len[r] = nn < 0 ? 0 : ok ? past + nn : past;
		s.q_start[r] = tok[r];
	}
	if (me == 0)
	{
		s.q_start[n] = tok[n];
		s.queue_out[0] = (head + taken) % np;
		s.queue_out[1] = count - taken + given;
		s.queue_out[2] = lack[n] - taken;
		s.queue_out[3] = tok[n];
	}
	for (int x = me; x < taken; x += step) // the new pages' entries
	{
		const int r = last_at_most(lack, n - 1, x);
		const int b = max(0, min(s.held[r], s.max_blocks)) + x - lack[r];
		s.block_table[(size_t)r * s.table_stride + b] = s.ring[(head + x) % np];
	}
	for (int x = me; x < given; x += step) // the returned pages, behind the free ones
	{
		const int r = last_at_most<SAT>(back, n - 1, x);
		s.ring[((long long)head + count + x) % np] = s.block_table[(size_t)r * s.table_stride + x - (back[r] & SAT)];
	}
	for (int t = me; t < s.max_tok; t += step)
	{
		int pos = 0, slot = -1, req = -1;
		if (t < tok[n])
		{
			req = last_at_most(tok, n - 1, t);
			const int held = max(0, min(s.held[req], s.max_blocks));
			pos = s.past[req] + t - tok[req];
			if (back[req + 1] & SERVED)
			{
				const int b = pos / s.page_size;
				const int page = b < held ? s.block_table[(size_t)req * s.table_stride + b]
				                          : s.ring[(head + lack[req] + b - held) % np];
				slot = page * s.page_size + pos % s.page_size;
			}
		}
		s.positions[t] = pos;
		s.slots[t] = slot;
		s.token_req[t] = req;
	}
}

// ---- norm and rotation by per-token positions ---------------------------------------
//
// Memory bound: 8 bytes a value. A CTA takes tokens in turn; a token's angles
// (their cosines and sines) serve all its heads, so they are formed once, in
// shared memory, while the first head vectors are already on their way, and
// then held in registers, as the gains are: a head vector is spread over LPV
// lanes, and a lane has the same places of every vector. Its item is the 2 VEC
// values that turn together (NEOX: VEC at e and VEC at e + n_rot / 2), so no
// exchange between lanes is needed but the norm's sum. 8192 tokens of 16/4
// heads x 256: 74 us, 4.6 TB/s (one CTA a token, gains and angles read for
// every vector: 85 us); 64 tokens of 32/8 x 128: 4.2 us. What is in flight runs
// out at a token's end: the next one's first loads follow this one's stores.

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_CTAS = 4 * 148; // what fits on the SMs at once: more tokens are taken in turn

struct RopeArgs
{
	nncu_rope_axes r;
	int half;
};

template <int VEC>
struct RopeVec
{
	float v[2 * VEC];
};

template <int VEC>
__device__ __forceinline__ void rope_load(RopeVec<VEC>& x, const float* p, int a, int b)
{
	if constexpr (VEC == 4)
	{
		const float4 u = *reinterpret_cast<const float4*>(p + a), w = *reinterpret_cast<const float4*>(p + b);
		x.v[0] = u.x, x.v[1] = u.y, x.v[2] = u.z, x.v[3] = u.w;
		x.v[4] = w.x, x.v[5] = w.y, x.v[6] = w.z, x.v[7] = w.w;
	}
	else
		x.v[0] = p[a], x.v[1] = p[b];
}

template <int VEC>
__device__ __forceinline__ void rope_store(const RopeVec<VEC>& x, float* p, int a, int b)
{
	if constexpr (VEC == 4)
	{
		*reinterpret_cast<float4*>(p + a) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
		*reinterpret_cast<float4*>(p + b) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
	}
	else
		p[a] = x.v[0], p[b] = x.v[1];
}

// IPL items a lane, LPV lanes a vector (a power of two).
template <int VEC, int IPL, int LPV, bool NEOX>
__global__ void __launch_bounds__(ROPE_THREADS, VEC * IPL <= 4 ? 4 : 2) rope_axes_kernel(const RopeArgs g)
{
	const nncu_rope_axes& r = g.r;
	__shared__ float2 turn[2][256]; // cos, sin of a token's pairs
	constexpr int VPC = ROPE_THREADS / LPV; // vectors in flight a CTA
	const int half = g.half, D = r.head_dim, items = D / (2 * VEC), turning = half / VEC;
	const int lane = threadIdx.x % LPV, slot = threadIdx.x / LPV;
	const int nq = r.q ? r.n_head : 0, n_vec = nq + (r.k ? r.n_kv : 0);

	// where this lane's items' two runs of VEC values begin (those past n_rot: two halves of the rest), and the gains
	int a[IPL], b[IPL];
	RopeVec<VEC> gq[IPL], gk[IPL];
#pragma unroll
	for (int j = 0; j < IPL; ++j)
	{
		const int i = lane + j * LPV;
		if (!NEOX)
			a[j] = 2 * VEC * i, b[j] = a[j] + VEC;
		else if (i < turning)
			a[j] = i * VEC, b[j] = a[j] + half;
		else
			a[j] = half + i * VEC, b[j] = a[j] + D / 2 - half;
#pragma unroll
		for (int e = 0; e < 2 * VEC; ++e) gq[j].v[e] = gk[j].v[e] = 1.0f;
		if (r.q_gamma && i < items) rope_load<VEC>(gq[j], r.q_gamma, a[j], b[j]);
		if (r.k_gamma && i < items) rope_load<VEC>(gk[j], r.k_gamma, a[j], b[j]);
	}
	const auto load = [&](RopeVec<VEC> (&x)[IPL], int t, int w) {
		const float* p = w < nq ? r.q + (size_t)t * r.q_stride + (size_t)w * D
		                        : r.k + (size_t)t * r.k_stride + (size_t)(w - nq) * D;
#pragma unroll
		for (int j = 0; j < IPL; ++j)
			if (lane + j * LPV < items) rope_load<VEC>(x[j], p, a[j], b[j]);
	};
	int buf = 0;
	for (int t = blockIdx.x; t < r.n_tok; t += gridDim.x, buf ^= 1)
	{
		RopeVec<VEC> x[IPL], ahead[IPL];
		int w = slot;
		if (w < n_vec) load(x, t, w);
		for (int i = threadIdx.x; i < half; i += ROPE_THREADS)
		{
			int axis = 0;
			if (r.interleaved)
			{
				const int m = i % r.n_axes;
				axis = i / r.n_axes < r.section[m] ? m : 0;
			}
			else
				for (int e = r.section[0]; axis + 1 < r.n_axes && i >= e; e += r.section[axis]) ++axis;
			const float angle = (float)r.positions[axis * r.pos_stride + t] * r.inv_freq[i];
			float sn, cs;
			sincosf(angle, &sn, &cs);
			turn[buf][i] = make_float2(cs, sn);
		}
		if (w + VPC < n_vec) load(ahead, t, w + VPC);
		__syncthreads(); // (two buffers: who comes here again has read this one long since)
		float2 cs[IPL][VEC];
#pragma unroll
		for (int j = 0; j < IPL; ++j)
#pragma unroll
			for (int e = 0; e < VEC; ++e)
				cs[j][e] = lane + j * LPV < turning ? turn[buf][(lane + j * LPV) * VEC + e] : make_float2(1.0f, 0.0f);

		for (; w < n_vec; w += VPC)
		{
			const bool is_q = w < nq;
			if (is_q ? r.q_gamma != nullptr : r.k_gamma != nullptr)
			{
				float ss = 0.0f;
#pragma unroll
				for (int j = 0; j < IPL; ++j)
					if (lane + j * LPV < items)
#pragma unroll
						for (int e = 0; e < 2 * VEC; ++e) ss = fmaf(x[j].v[e], x[j].v[e], ss);
				// the lanes of one vector leave the loop together, so they name each other alone
				const unsigned mask = LPV == 32 ? 0xffffffffu
				                                : ((1u << (LPV & 31)) - 1u) << ((threadIdx.x & 31) / LPV * LPV);
#pragma unroll
				for (int o = LPV / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
				const float sc = 1.0f / sqrtf(ss / (float)D + r.eps);
#pragma unroll
				for (int j = 0; j < IPL; ++j)
#pragma unroll
					for (int e = 0; e < 2 * VEC; ++e) x[j].v[e] = x[j].v[e] * sc * (is_q ? gq[j].v[e] : gk[j].v[e]);
			}
			float* y = is_q ? r.q_out + (size_t)t * r.q_out_stride + (size_t)w * D
			                : r.k_out + (size_t)t * r.k_out_stride + (size_t)(w - nq) * D;
#pragma unroll
			for (int j = 0; j < IPL; ++j)
			{
				if (lane + j * LPV >= items) continue;
				if (lane + j * LPV < turning)
				{
#pragma unroll
					for (int e = 0; e < VEC; ++e)
					{
						// NEOX: values e and e + VEC of the item; NORM: 2e and 2e + 1
						float& u = x[j].v[NEOX ? e : 2 * e];
						float& v = x[j].v[NEOX ? e + VEC : 2 * e + 1];
						const float u0 = u, v0 = v;
						u = u0 * cs[j][e].x - v0 * cs[j][e].y;
						v = u0 * cs[j][e].y + v0 * cs[j][e].x;
					}
				}
				rope_store<VEC>(x[j], y, a[j], b[j]);
			}
#pragma unroll
			for (int j = 0; j < IPL; ++j) x[j] = ahead[j];
			if (w + 2 * VPC < n_vec) load(ahead, t, w + 2 * VPC);
		}
	}
}

template <int VEC, int IPL, int LPV>
void launch_rope_as(const RopeArgs& g, cudaStream_t st)
{
	const unsigned grid = (unsigned)(g.r.n_tok < ROPE_CTAS ? g.r.n_tok : ROPE_CTAS);
	if (g.r.rope_mode == NNCU_ROPE_NEOX)
		rope_axes_kernel<VEC, IPL, LPV, true><<<grid, ROPE_THREADS, 0, st>>>(g);
	else
		rope_axes_kernel<VEC, IPL, LPV, false><<<grid, ROPE_THREADS, 0, st>>>(g);
}

template <int VEC>
int launch_rope_axes(const RopeArgs& g, cudaStream_t st)
{
	const int items = g.r.head_dim / (2 * VEC);
	if (items <= 8)
		launch_rope_as<VEC, 1, 8>(g, st);
	else if (items <= 16)
		launch_rope_as<VEC, 1, 16>(g, st);
	else if (items <= 32)
		launch_rope_as<VEC, 1, 32>(g, st);
	else if (items <= 64)
		launch_rope_as<VEC, 2, 32>(g, st);
	else if (VEC == 1)
		launch_rope_as<1, 8, 32>(g, st);
	note_launches(1);
	return (int)cudaGetLastError();
}

// ---- the 4-bit cache's write -----------------------------------------------------------
//
// 4 bytes a value in, 0.5625 out. A lane takes 8 values, which become one
// 32-bit word, four lanes a group of 32: its largest magnitude (with its sign as
// the lowest bit, so that the positive one wins a tie) meets in two exchanges,
// and every lane forms the scale and its reciprocal. blockIdx.y: K or V. 8191
// tokens of 4 heads x 256, written and read back: 45 us, 3.4 TB/s (four values a
// lane and three exchanges of three values: 60 us). 16384 tokens: the write 41
// us, 3.7 TB/s, bound by loads in flight and issue slots (70 % busy); the read 50
// us, 3.1 TB/s, bound by the load and store path (L1 87 % busy). Every thread
// also copies its parameters, which it indexes by K or V, to local memory.

constexpr int ROWS_THREADS = 256;
constexpr int ROWS_ITEMS = 2;           // pieces (8 values, 32 bytes) in flight a thread
constexpr long long ROWS_MOST = 1 << 30; // pieces of one launch, so that 32 bits number them

struct RowsArgs
{
	uint8_t* pages;
	int n_pages, page_shift, n_kv, d_shift, n_tok;
	uint32_t per_tok;  // pieces of 8 values a token
	uint32_t div_m;    // piece / per_tok = piece * div_m >> div_s (pieces below 2^31)
	int div_s;
	const int* slots;
	float* x[2];
	size_t stride[2];
	int first; // 0: from K; 1: V only
};

// Piece i: its token, and the piece within the token's row.
__device__ __forceinline__ void rows_split(const RowsArgs& a, uint32_t i, uint32_t& t, uint32_t& piece)
{
	t = (uint32_t)(((uint64_t)i * a.div_m) >> a.div_s);
	piece = i - t * a.per_tok;
}

// Where a token's row of one KV head sits: its codes and its scales.
__device__ __forceinline__ bool rows_at(const RowsArgs& a, int which, int slot, int h, int& off, uint8_t*& codes,
                                        uint16_t*& scales)
{
	const int pg = slot >> a.page_shift, page = 1 << a.page_shift, D = 1 << a.d_shift;
	if (slot < 0 || pg >= a.n_pages) return false;
	off = slot & (page - 1);
	const int cb = kv4_codes_bytes(page, D), sb = kv4_scales_bytes(page, D);
	uint8_t* chunk = a.pages + ((size_t)pg * a.n_kv + h) * kv4_chunk_bytes(page, D);
	codes = chunk + which * cb + off * (D / 2);
	scales = reinterpret_cast<uint16_t*>(chunk + 2 * cb + which * sb) + off * (D / KV4_GROUP);
	return true;
}

__global__ void __launch_bounds__(ROWS_THREADS) kv4_append_kernel(const RowsArgs a)
{
	const int which = a.first + blockIdx.y, D = 1 << a.d_shift;
	const float* __restrict__ src = a.x[which]; // (K and V rows are read, never written)
	const size_t stride = a.stride[which];
	const uint32_t total = (uint32_t)a.n_tok * a.per_tok;
	const uint32_t base = blockIdx.x * (ROWS_THREADS * ROWS_ITEMS) + threadIdx.x;
	float x[ROWS_ITEMS][8];
	int slot[ROWS_ITEMS];
	uint32_t piece[ROWS_ITEMS];
#pragma unroll
	for (int j = 0; j < ROWS_ITEMS; ++j)
	{
		const uint32_t i = base + j * ROWS_THREADS;
		slot[j] = -1;
		piece[j] = 0;
		float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f), w = v;
		if (i < total)
		{
			uint32_t t;
			rows_split(a, i, t, piece[j]);
			slot[j] = a.slots[t];
			const float4* p = reinterpret_cast<const float4*>(src + (size_t)t * stride + 8 * (size_t)piece[j]);
			v = __ldcs(p);
			w = __ldcs(p + 1);
		}
		x[j][0] = v.x, x[j][1] = v.y, x[j][2] = v.z, x[j][3] = v.w;
		x[j][4] = w.x, x[j][5] = w.y, x[j][6] = w.z, x[j][7] = w.w;
	}
#pragma unroll
	for (int j = 0; j < ROWS_ITEMS; ++j)
	{
		// (whole warps: a group's 4 lanes always work on one row)
		uint32_t top = 0; // magnitude's bits, then 1 where positive
#pragma unroll
		for (int e = 0; e < 8; ++e)
		{
			const uint32_t u = __float_as_uint(x[j][e]);
			top = max(top, (u << 1) | (~u >> 31));
		}
		top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
		top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
		const bool bad = (top >> 1) >= 0x7f800000u; // an infinity or a NaN
		const float m = __uint_as_float((top >> 1) | (~top << 31));
		float s = __bfloat162float(__float2bfloat16_rn(m * -0.125f));
		s = copysignf(fminf(fmaxf(fabsf(s), KV4_SCALE_MIN), KV4_SCALE_MAX), s);
		const float inv = __frcp_rn(s);
		uint32_t c[8]; // code + 8 in the low bits: the sum rounds to the nearest whole number, ties to even
#pragma unroll
		for (int e = 0; e < 8; ++e)
			c[e] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x[j][e], inv), -8.0f), 7.0f), 12582920.0f)) & 15u;
		uint32_t w = 0;
#pragma unroll
		for (int e = 0; e < 8; ++e) w |= c[e] << (4 * kv4_nibble(e));
		if (bad) w = 0x88888888u;
		const int h = piece[j] >> (a.d_shift - 3), in = piece[j] & (D / 8 - 1), g = in / 4;
		int off;
		uint8_t* codes;
		uint16_t* scales;
		if (rows_at(a, which, slot[j], h, off, codes, scales))
		{
			*reinterpret_cast<uint32_t*>(codes + 16 * kv4_unit(off, g, D) + 4 * (in & 3)) = w;
			if ((in & 3) == 0) scales[g] = bad ? (uint16_t)0x7fc0u : (uint16_t)(__float_as_uint(s) >> 16);
		}
	}
}

// ---- and its reading back: a piece is a word --------------------------------------------

__global__ void __launch_bounds__(ROWS_THREADS) kv4_read_kernel(const RowsArgs a)
{
	const int which = a.first + blockIdx.y, D = 1 << a.d_shift;
	const uint32_t total = (uint32_t)a.n_tok * a.per_tok;
	const uint32_t base = blockIdx.x * (ROWS_THREADS * ROWS_ITEMS) + threadIdx.x;
	uint32_t t[ROWS_ITEMS], piece[ROWS_ITEMS], w[ROWS_ITEMS];
	int slot[ROWS_ITEMS];
	float s[ROWS_ITEMS];
#pragma unroll
	for (int j = 0; j < ROWS_ITEMS; ++j)
	{
		const uint32_t i = base + j * ROWS_THREADS;
		rows_split(a, i < total ? i : 0, t[j], piece[j]);
		slot[j] = a.slots[t[j]];
	}
#pragma unroll
	for (int j = 0; j < ROWS_ITEMS; ++j)
	{
		const int h = piece[j] >> (a.d_shift - 3), in = piece[j] & (D / 8 - 1), g = in / 4;
		int off;
		uint8_t* codes;
		uint16_t* scales;
		w[j] = 0;
		s[j] = 0.0f;
		if (rows_at(a, which, slot[j], h, off, codes, scales))
		{
			w[j] = *reinterpret_cast<const uint32_t*>(codes + 16 * kv4_unit(off, g, D) + 4 * (in & 3));
			s[j] = bf16_bits_to_float(scales[g]);
		}
	}
#pragma unroll
	for (int j = 0; j < ROWS_ITEMS; ++j)
	{
		if (base + j * ROWS_THREADS >= total) continue;
		float y[8];
#pragma unroll
		for (int e = 0; e < 8; ++e)
			y[e] = s[j] * (__uint_as_float(((w[j] >> (4 * kv4_nibble(e))) & 15u) | 0x4b000000u) - 8388616.0f); // 2^23 + u, less 2^23 + 8
		float4* p = reinterpret_cast<float4*>(a.x[which] + (size_t)t[j] * a.stride[which] + 8 * (size_t)piece[j]);
		__stcs(p, make_float4(y[0], y[1], y[2], y[3]));
		__stcs(p + 1, make_float4(y[4], y[5], y[6], y[7]));
	}
}

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks of a rows call; 1: nothing to do.
int rows_args(const nncu_kv4_rows* r, const char* what, RowsArgs& a)
{
	char msg[160];
	if (!r) return refuse("kv4 rows: NULL argument");
	const int rc = kv4_check_pool(&r->pool, what);
	if (rc != NNCU_OK) return rc;
	const size_t row = (size_t)r->pool.n_kv * r->pool.head_dim;
	msg[0] = 0;
	if (r->n_tok < 0)
		snprintf(msg, sizeof msg, "%s: negative n_tok", what);
	else if (r->n_tok > 0 && (!r->slots || (!r->k && !r->v)))
		snprintf(msg, sizeof msg, "%s: NULL slots or rows", what);
	else if (!aligned16(r->k) || !aligned16(r->v) || (r->k && r->k_stride % 4) || (r->v && r->v_stride % 4))
		snprintf(msg, sizeof msg, "%s: rows must be 16-byte aligned", what);
	else if (r->n_tok > 1 && ((r->k && r->k_stride < row) || (r->v && r->v_stride < row)))
		snprintf(msg, sizeof msg, "%s: strides shorter than a row", what);
	if (msg[0]) return refuse(msg);
	const auto log2i = [](int x) {
		int s = 0;
		while ((1 << s) < x) ++s;
		return s;
	};
	const uint32_t per_tok = (uint32_t)(row / 8);
	int s = 0; // ceil(log2 per_tok): the multiplier 2^(31 + s) / per_tok, rounded up, fits 32 bits and divides exactly
	while ((1ull << s) < per_tok) ++s;
	a = RowsArgs{static_cast<uint8_t*>(r->pool.pages), r->pool.n_pages, log2i(r->pool.page_size), r->pool.n_kv,
	             log2i(r->pool.head_dim), r->n_tok, per_tok, (uint32_t)(((1ull << (31 + s)) + per_tok - 1) / per_tok),
	             31 + s, r->slots, {r->k, r->v}, {r->k_stride, r->v_stride}, r->k ? 0 : 1};
	return NNCU_OK;
}

// The rows in launches of at most ROWS_MOST pieces.
template <typename K>
int launch_rows(K kernel, RowsArgs a, cudaStream_t st)
{
	const int most = (int)(ROWS_MOST / a.per_tok), all = a.n_tok;
	for (int t0 = 0; t0 < all; t0 += most)
	{
		a.n_tok = all - t0 < most ? all - t0 : most;
		const uint32_t pieces = (uint32_t)a.n_tok * a.per_tok;
		const dim3 grid((pieces + ROWS_THREADS * ROWS_ITEMS - 1) / (ROWS_THREADS * ROWS_ITEMS), a.x[0] && a.x[1] ? 2u : 1u);
		kernel<<<grid, ROWS_THREADS, 0, st>>>(a);
		note_launches(1);
		a.slots += a.n_tok;
		for (int w = 0; w < 2; ++w)
			if (a.x[w]) a.x[w] += (size_t)a.n_tok * a.stride[w];
	}
	return (int)cudaGetLastError();
}

} // namespace

int kv4_check_pool(const nncu_kv4_pool* p, const char* what, bool need_pages)
{
	char msg[160];
	msg[0] = 0;
	if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
		snprintf(msg, sizeof msg, "%s: head_dim %d (64, 128 and 256 are served)", what, (int)p->head_dim);
	else if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
		snprintf(msg, sizeof msg, "%s: page_size %d (16, 32, 64, 128 or 256)", what, (int)p->page_size);
	else if (p->n_pages <= 0 || p->n_kv <= 0 || (long long)p->n_pages * p->page_size > INT32_MAX || (long long)p->n_kv * p->head_dim > (1 << 24))
		snprintf(msg, sizeof msg, "%s: bad n_pages or n_kv", what);
	else if (need_pages && (!p->pages || !aligned16(p->pages)))
		snprintf(msg, sizeof msg, "%s: pages NULL or not 16-byte aligned", what);
	return msg[0] ? refuse(msg) : NNCU_OK;
}

} // namespace nncu

using namespace nncu;

namespace
{

// Whether an array that a step writes shares entries with another of its arrays: CTAs read and write them at the same
// time.
bool step_arrays_meet(const nncu_paged_step& s)
{
	struct Array
	{
		const int32_t* p;
		size_t n;
	};
	const size_t n = s.n_req, tok = s.max_tok;
	const Array all[] = {{s.held_out, n},  {s.queue_out, 4}, {s.seq_len, n},   {s.q_start, n + 1},          {s.positions, tok},
	                     {s.slots, tok},   {s.token_req, tok}, {s.ring, (size_t)s.n_pages}, // written, the ones below only read
	                     {s.past, n},      {s.n_new, n},     {s.held, n},      {s.queue, 2}};
	constexpr int ALL = sizeof all / sizeof all[0], WRITTEN = 8;
	const auto at = [](const int32_t* p) { return reinterpret_cast<uintptr_t>(p); };
	const uintptr_t table = at(s.block_table), row = 4 * (uintptr_t)s.table_stride;
	for (int i = 0; i < ALL; ++i)
	{
		const uintptr_t p = at(all[i].p), e = p + 4 * all[i].n;
		if (p == e) continue;
		for (int j = 0; j < i && j < WRITTEN; ++j)
			if (p < at(all[j].p + all[j].n) && at(all[j].p) < e) return true;
		// the table's rows, without what lies between them
		if (e <= table || p >= table + (n - 1) * row + 4 * (uintptr_t)s.max_blocks) continue;
		if (p < table || (p - table) % row < 4 * (uintptr_t)s.max_blocks || (p - table) % row + (e - p) > row) return true;
	}
	return false;
}

} // namespace

extern "C" int nncu_paged_step_dev(const nncu_paged_step* s, void* stream)
{
	if (!s) return refuse("paged step: NULL argument");
	if (s->n_req <= 0 || s->n_req > NNCU_PAGED_MAX_REQ) return refuse("paged step: n_req out of range");
	if (s->page_size <= 0 || s->n_pages <= 0 || s->max_blocks <= 0 || s->max_tok < 0 || s->max_tok > (1 << 28) ||
	    (long long)s->n_pages * s->page_size > INT32_MAX || (long long)s->max_blocks * s->page_size > INT32_MAX ||
	    s->n_pages > (1 << 29))
		return refuse("paged step: bad page_size, n_pages, max_blocks or max_tok");
	if (s->table_stride < s->max_blocks) return refuse("paged step: table rows shorter than max_blocks");
	if (!s->past || !s->n_new || !s->held || !s->queue || !s->ring || !s->block_table || !s->held_out ||
	    !s->queue_out || !s->seq_len || !s->q_start || (s->max_tok > 0 && (!s->positions || !s->slots || !s->token_req)))
		return refuse("paged step: NULL array");
	if (s->held_out == s->held || s->queue_out == s->queue)
		return refuse("paged step: held_out and queue_out must not be the inputs");
	if (step_arrays_meet(*s)) return refuse("paged step: an array that is written must not meet another one");
	const size_t smem = 3 * sizeof(int) * ((size_t)s->n_req + 1);
	if (smem + STEP_WARPS * sizeof(int) > 48 * 1024) // what a kernel has unasked, its fixed arrays included
	{
		const cudaError_t ce = cudaFuncSetAttribute(paged_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
		                                            3 * (int)sizeof(int) * (NNCU_PAGED_MAX_REQ + 1));
		if (ce != cudaSuccess) return set_cuda_error((int)ce, "paged step shared memory");
	}
	// four tokens a thread; every CTA repeats the sums, so no more than that asks for
	const int work = s->max_tok > s->n_req ? s->max_tok : s->n_req;
	const int grid = (work + 4 * STEP_THREADS - 1) / (4 * STEP_THREADS);
	paged_step_kernel<<<grid < 296 ? grid : 296, STEP_THREADS, smem, static_cast<cudaStream_t>(stream)>>>(*s);
	note_launches(1);
	const int e = (int)cudaGetLastError();
	return e ? set_cuda_error(e, "paged step launch") : NNCU_OK;
}

extern "C" int nncu_rope_axes_dev(const nncu_rope_axes* r, void* stream)
{
	if (!r) return refuse("rope axes: NULL argument");
	if (r->n_tok < 0 || (!r->q && !r->k)) return refuse("rope axes: negative n_tok or no rows");
	if (r->n_tok > INT32_MAX - ROPE_CTAS) return refuse("rope axes: n_tok too large"); // (the CTAs count past it by that many)
	if (r->head_dim <= 0 || r->head_dim > 512 || r->head_dim % 2) return refuse("rope axes: head_dim must be even, up to 512");
	if (r->n_rot < 0 || r->n_rot % 2 || r->n_rot > r->head_dim) return refuse("rope axes: n_rot must be even, up to head_dim");
	if (r->rope_mode != NNCU_ROPE_NEOX && r->rope_mode != NNCU_ROPE_NORM) return refuse("rope axes: unknown rope mode");
	if (r->n_axes < 1 || r->n_axes > 4) return refuse("rope axes: one to four axes");
	long long pairs = 0;
	for (int a = 0; a < r->n_axes; ++a)
	{
		if (r->section[a] < 0) return refuse("rope axes: negative section");
		pairs += r->section[a];
	}
	if (pairs != r->n_rot / 2) return refuse("rope axes: the sections must have n_rot / 2 pairs together");
	if (r->interleaved)
		for (int a = 1; a < r->n_axes; ++a)
			if (r->section[a] > 0 && (long long)(r->section[a] - 1) * r->n_axes + a >= r->n_rot / 2)
				return refuse("rope axes: an interleaved section passes the last pair");
	if ((r->q && (!r->q_out || r->n_head <= 0)) || (r->k && (!r->k_out || r->n_kv <= 0)))
		return refuse("rope axes: NULL output or no heads");
	if (r->n_rot > 0 && (!r->positions || !r->inv_freq)) return refuse("rope axes: NULL positions or frequencies");
	if (r->n_tok > 1 && r->n_axes > 1 && r->pos_stride < (size_t)r->n_tok)
		return refuse("rope axes: pos_stride shorter than the tokens");
	const size_t qrow = (size_t)r->n_head * r->head_dim, krow = (size_t)r->n_kv * r->head_dim;
	if (r->n_tok > 1 && ((r->q && (r->q_stride < qrow || r->q_out_stride < qrow)) ||
	                     (r->k && (r->k_stride < krow || r->k_out_stride < krow))))
		return refuse("rope axes: strides shorter than a row");
	if ((r->q && r->q == r->q_out && r->q_stride != r->q_out_stride) ||
	    (r->k && r->k == r->k_out && r->k_stride != r->k_out_stride))
		return refuse("rope axes: in place with two strides");
	if (r->n_tok == 0) return NNCU_OK;
	const RopeArgs g{*r, r->n_rot / 2};
	// 16-byte accesses where every run of four values allows them
	const bool vec = r->head_dim % 8 == 0 && r->n_rot % 8 == 0 && aligned16(r->q) && aligned16(r->k) &&
	                 aligned16(r->q_out) && aligned16(r->k_out) && aligned16(r->q_gamma) && aligned16(r->k_gamma) &&
	                 (!r->q || (r->q_stride % 4 == 0 && r->q_out_stride % 4 == 0)) &&
	                 (!r->k || (r->k_stride % 4 == 0 && r->k_out_stride % 4 == 0));
	const auto st = static_cast<cudaStream_t>(stream);
	const int e = vec ? launch_rope_axes<4>(g, st) : launch_rope_axes<1>(g, st);
	return e ? set_cuda_error(e, "rope axes launch") : NNCU_OK;
}

extern "C" int nncu_kv4_bytes(const nncu_kv4_pool* pool, size_t* bytes)
{
	if (!pool || !bytes) return refuse("kv4 bytes: NULL argument");
	const int rc = kv4_check_pool(pool, "kv4 bytes", false);
	if (rc != NNCU_OK) return rc;
	*bytes = kv4_chunk_bytes(pool->page_size, pool->head_dim) * pool->n_kv * pool->n_pages;
	return NNCU_OK;
}

extern "C" int nncu_kv4_append_dev(const nncu_kv4_rows* rows, void* stream)
{
	RowsArgs a;
	const int rc = rows_args(rows, "kv4 append", a);
	if (rc != NNCU_OK || a.n_tok == 0) return rc;
	const int e = launch_rows(kv4_append_kernel, a, static_cast<cudaStream_t>(stream));
	return e ? set_cuda_error(e, "kv4 append launch") : NNCU_OK;
}

extern "C" int nncu_kv4_read_dev(const nncu_kv4_rows* rows, void* stream)
{
	RowsArgs a;
	const int rc = rows_args(rows, "kv4 read", a);
	if (rc != NNCU_OK || a.n_tok == 0) return rc;
	const int e = launch_rows(kv4_read_kernel, a, static_cast<cudaStream_t>(stream));
	return e ? set_cuda_error(e, "kv4 read launch") : NNCU_OK;
}
