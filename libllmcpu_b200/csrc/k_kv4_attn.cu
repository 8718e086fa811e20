// k_kv4_attn.cu -- attention of packed requests over the paged 4-bit cache
// (nncu_kv4_attention_dev): the entry, and the kernel for requests with few
// query rows (decode, verify; prompts: k_kv4_prompt.cu).
//
// Work. A segment is (request, KV head, row group): 8 R query rows (token x
// grouped head) that read the same keys. Its keys are walked in tiles of 64;
// the segments' tiles, one request after another, are cut into equal runs,
// one per CTA, whatever the requests' lengths: every CTA finds its run from
// the lengths on the device (a scan over the requests), so one launch serves
// any batch and a captured graph follows new lengths. A run is a few pieces of
// segments; a piece that is a whole segment writes the output, another leaves
// its unnormalised sum with its maximum and weight in the workspace, and the
// CTA that adds the last piece of a segment joins them in order.
//
// A CTA is four computing warps, 16 keys of a tile each, with a softmax state
// of their own until the piece's end, and one warp that keeps a ring of tiles
// coming (bulk copies of the pages' codes and scales, looked up in the block
// table 32 entries at a time).
//
// Mathematics. For a group of 32 values (one scale s) q.k = s sum q c: the
// codes c go to the tensor cores unscaled (a mask and a subtraction make them
// 16-bit floats) and the group's sum takes its scale in 32 bits. V's codes
// cannot wait for their scale (the sum runs over keys), but 8 bits of scale
// times 4 of code are exact in a 16-bit float. q and the weights p go in as
// two 16-bit halves each (22 bits), accumulated in 32: the result is as close
// to the exact one as 32-bit arithmetic. (Codes as denormal floats, straight
// from a mask, would save the subtraction, but the products' adder aligns by
// exponents and cuts off the bits that the denormals lack: 3e-6 instead of
// 1e-6 of the output.)
// What bounds it: issue slots, about 470 instructions per 16 keys of 128
// values (150 of them unpack), and pieces' starts and ends (a third of the
// cycles), not memory. 64 requests of 512 to 8192 keys, 32/8 heads x 128: 93
// us, 2.24 TB/s of the cache; 131072 keys, 8/4 x 256, four tokens: 89 us, 1.7
// TB/s; 4096 keys, 32/8 x 128: 16 us (latency).
// Requests with many query rows a KV head (few_rows) are left to the
// tensor-memory kernel: it takes 128 rows or more at a time for the price of
// one unpacking, this one 8 to 32.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cmath>
#include <cstdio>

#include "kv4.cuh"

namespace nncu
{
namespace
{

constexpr int TILE = 64;               // keys a tile
constexpr int CW = 4;                  // computing warps, 16 keys of a tile each
constexpr int THREADS = (CW + 1) * 32; // and the loading warp
constexpr int STAGES = 3;              // tiles in the ring: what arrives while one is worked on
// Requests with more query rows a KV head go to k_kv4_prompt.cu. Measured, 16
// requests over 4000 keys, 8 KV heads (256: 4), here and there: 64 values a
// head, 128 rows 181 and 212 us; 128, 96 rows 259 and 361, 128 rows 339 and
// 293; 256, 64 rows 221 and 246, 96 rows 325 and 249. With few key tiles (one
// request: 250 to 500 of them), where more and shorter pieces are what counts,
// twice as many stay here: 128, 128 rows 41 and 72 us; 256, 128 rows 42 and 77.
constexpr int few_rows(int D) { return D == 64 ? 128 : D == 128 ? 96 : 64; }
// Several row tiles a segment share the unpacking, single ones make more and
// shorter segments: 16 requests over 4000 keys, 8 KV heads x 128, 32 rows, two
// tiles 101 us, one 118; one request, two 34 us, one 24. So several from this
// many key tiles on. (The most that the tables can hold, the lengths being on
// the device: one request over 4000 keys with a table for 131072 takes two row
// tiles, 34 us, and with 128 rows the other kernel, 66 us instead of 41.)
constexpr long long MANY_TILES = 4096, FEW_TILES = 1024;
constexpr int MIN_TILES = 4;           // a run is at least this long, while tiles are few
// A row's weights are taken against a held score, 2^11 at it, which moves only
// when a score passes it by more than 2^4: then no weight passes 2^15, within a
// 16-bit float, and weights of 2^-24 of the largest keep 11 bits and more.
constexpr float P_SCALE = 11.0f, P_TOP = 15.0f;
constexpr float NONE = 1e30f; // P_SCALE - held score of a row that has seen no key yet

// What a launch keeps in the workspace: an error word, a counter per CTA (of
// the segment that begins in the CTA's run and does not end there), and two
// partial results per CTA (of its first and its last piece).
struct Ws
{
	int* err;
	int* counters;
	float* parts;
};

template <int D, int R>
struct Shape
{
	static constexpr int U = D / KV4_GROUP, ROWS = 8 * R;
	static constexpr int CODES = TILE * D / 2, SCALES = TILE * U * 2;
	static constexpr int STAGE = 2 * (CODES + SCALES);
	static constexpr int RED_ROW = D + 4;                   // floats a row of the joining buffer
	static constexpr int SM_RED = STAGES * STAGE;           // [CW][ROWS][RED_ROW]
	static constexpr int SM_Q = SM_RED + CW * ROWS * RED_ROW * 4; // q's operands [D / 16][R][32 lanes] of 16 bytes
	static constexpr int SM_ML = SM_Q + D / 16 * R * 512;   // [CW][ROWS] (maximum, weight)
	static constexpr int SM_BAR = SM_ML + CW * ROWS * 8;
	static constexpr int SMEM = SM_BAR + 256;
	static_assert(SM_BAR % 16 == 0 && SM_Q % 16 == 0 && SM_RED % 16 == 0 && SCALES % 16 == 0, "aligned for their accesses");
	static_assert(2 * STAGES * 8 + (STAGES + 2) * 4 <= 128, "barriers and words before the scan");
	static constexpr int PART = ROWS * (D + 2);             // floats a partial result
	static constexpr int CTAS = D * R <= 128 ? 4 : D == 256 ? 2 : 3; // per SM
	static_assert(192 * CTAS * 4 <= 4096, "a counter per CTA");
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
	asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
	    : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
	    : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from nothing: d = A B.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1)
{
	asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
	    : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
	    : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// An 8 x 8 matrix of 16-bit values, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
	uint32_t y;
	asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
	return y;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// x, y as 16-bit halves: hi the rounded values, lo what they leave.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo)
{
	const __half2 h = __floats2half2_rn(x, y);
	const float2 f = __half22float2(h);
	hi = half2_bits(h);
	lo = half2_bits(__floats2half2_rn(x - f.x, y - f.y));
}

// N neighbouring scales.
template <int N>
__device__ __forceinline__ void load_scales(float (&f)[N], const unsigned char* p)
{
	if constexpr (N == 1)
		f[0] = bf16_bits_to_float(*reinterpret_cast<const uint16_t*>(p));
	else
	{
		uint32_t w[N / 2];
		if constexpr (N == 2)
			w[0] = *reinterpret_cast<const uint32_t*>(p);
		else if constexpr (N == 4)
		{
			const uint2 x = *reinterpret_cast<const uint2*>(p);
			w[0] = x.x, w[1] = x.y;
		}
		else
		{
			const uint4 x = *reinterpret_cast<const uint4*>(p);
			w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
		}
#pragma unroll
		for (int i = 0; i < N / 2; ++i)
			f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
	}
}

// Nibbles x and x + 4 of a word as codes: the mask makes 1024 + u (or 64 + u,
// one nibble up) in the two halves, less 1032 (72): exact.
struct Masks
{
	uint32_t low = 0x000F000Fu, high = 0x00F000F0u, k1024 = 0x64006400u, k64 = 0x54005400u;
	// kept in registers: as constants, one of the two that an operation needs would be moved there every time
	__device__ __forceinline__ Masks() { asm volatile("" : "+r"(low), "+r"(high), "+r"(k1024), "+r"(k64)); }
};
__device__ __forceinline__ __half2 codes2(const Masks& mk, uint32_t w, int x)
{
	const uint32_t v = x >= 2 ? w >> 8 : w;
	const uint32_t h = x & 1 ? (v & mk.high) | mk.k64 : (v & mk.low) | mk.k1024;
	return __hadd2(bits_half2(h), __float2half2_rn(x & 1 ? -72.0f : -1032.0f));
}

// One segment's rows and the tiles of its keys.
struct Segment
{
	Kv4Request x;
	int r, hk, row0, rows;   // request, KV head, first row of the group, rows of the request (token x grouped head)
	int tile0, tiles;        // first tile and their number, for every segment of the request
	int first, last;         // keys of the request's new tokens together
};

__device__ __forceinline__ void segment_tiles(const Kv4Args& a, Segment& s, int r)
{
	s.r = r;
	s.x = kv4_request(a, r);
	s.rows = s.x.n_new * a.group;
	if (s.rows > a.few_rows) s.rows = 0; // the tensor-memory kernel's
	s.last = min(s.x.pos0 + s.x.n_new - 1, s.x.keys - 1);
	s.first = kv4_first_key(a, s.x.pos0);
	s.tile0 = s.first / TILE;
	s.tiles = s.rows == 0 ? 0 : s.last < s.first ? 1 : s.last / TILE - s.tile0 + 1;
}

// Equal runs of `total` tiles over n CTAs: the first total % n one longer.
struct Runs
{
	long long per, rem;
	__device__ __forceinline__ long long begin(int c) const { return c * per + min((long long)c, rem); }
	__device__ __forceinline__ int owner(long long t) const
	{
		const long long u = t - rem * (per + 1); // behind the longer runs
		const long long x = u < 0 ? t : u, d = u < 0 ? per + 1 : per;
		const int q = ((x | d) >> 32) == 0 ? (int)((uint32_t)x / (uint32_t)d) : (int)(x / d);
		return u < 0 ? q : (int)rem + q;
	}
};

template <int D, int R>
__global__ void __launch_bounds__(THREADS, (Shape<D, R>::CTAS)) kv4_decode_kernel(const Kv4Args a, const Ws ws)
{
	using L = Shape<D, R>;
	constexpr int U = L::U, J = U / 2, ROWS = L::ROWS;
	extern __shared__ __align__(128) unsigned char smem[];
	float* red = reinterpret_cast<float*>(smem + L::SM_RED);
	uint4* qsm = reinterpret_cast<uint4*>(smem + L::SM_Q);
	float2* ml = reinterpret_cast<float2*>(smem + L::SM_ML);
	uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::SM_BAR);
	uint64_t* empty = full + STAGES;
	int* loaded = reinterpret_cast<int*>(empty + STAGES); // [STAGES]: which 16-key parts of the tile came
	volatile int* abort_ = loaded + STAGES;
	int* last_piece = loaded + STAGES + 1;
	long long* scan = reinterpret_cast<long long*>(smem + L::SM_BAR + 128); // warp sums, then the start
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

	if (tid == 0)
	{
		for (int s = 0; s < STAGES; ++s)
		{
			mbar_init(&full[s], 1);
			mbar_init(&empty[s], CW);
		}
		*abort_ = 0;
		fence_barrier_init();
	}

	// ---- this CTA's run: a scan of the requests' tiles, each thread a few requests ----
	const int each = (a.n_req + THREADS - 1) / THREADS;
	const auto cost = [&](const Segment& s) {
		return (long long)s.tiles * a.n_kv * ((s.rows + ROWS - 1) / ROWS);
	};
	long long mine = 0;
	for (int r = tid * each; r < min(a.n_req, (tid + 1) * each); ++r)
	{
		Segment s;
		segment_tiles(a, s, r);
		mine += cost(s);
	}
	long long before = mine;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1)
	{
		const long long u = __shfl_up_sync(0xffffffffu, before, o);
		if (lane >= o) before += u;
	}
	if (lane == 31) scan[warp] = before;
	__syncthreads();
	long long total = 0;
	before -= mine;
	for (int w = 0; w <= CW; ++w)
	{
		if (w < warp) before += scan[w];
		total += scan[w];
	}
	const int n_ctas = (int)min((long long)gridDim.x, max(1ll, total / MIN_TILES));
	const Runs runs{total / n_ctas, total % n_ctas};
	if ((int)blockIdx.x >= n_ctas || total == 0) return;
	const long long run0 = runs.begin(blockIdx.x);
	__syncthreads();
	if (before <= run0 && run0 < before + mine)
	{
		long long at = before;
		for (int r = tid * each;; ++r)
		{
			Segment s;
			segment_tiles(a, s, r);
			const long long c = cost(s);
			if (run0 < at + c)
			{
				scan[0] = r;
				scan[1] = run0 - at;
				break;
			}
			at += c;
		}
	}
	__syncthreads();
	const int start_req = (int)scan[0];
	const long long start_off = scan[1];
	int left = (int)(runs.begin(blockIdx.x + 1) - run0);

	// the pieces of the run, one after another (the same for every warp)
	Segment s;
	segment_tiles(a, s, start_req);
	int groups = (s.rows + ROWS - 1) / ROWS;
	int seg = (int)(start_off / s.tiles), tile = (int)(start_off % s.tiles); // segment of the request, tile of the segment
	long long seg_at = run0 - tile;                                          // the segment's first tile among all
	const auto next_piece = [&](int done) {
		left -= done;
		seg_at += s.tiles;
		tile = 0;
		if (left > 0 && ++seg == a.n_kv * groups)
		{
			seg = 0;
			int r = s.r;
			do segment_tiles(a, s, ++r);
			while (s.rows == 0);
			groups = (s.rows + ROWS - 1) / ROWS;
		}
	};

	if (warp == CW)
	{
		// ---- the loading warp: lane = 4 x part of the tile + {K codes, V codes, K scales, V scales} ----
		const int parts = min(TILE, a.page), n_parts = TILE / parts; // keys a part, parts a tile
		const int what = lane & 3, part = lane >> 2;
		const int cb = kv4_codes_bytes(a.page, D), sb = kv4_scales_bytes(a.page, D);
		const uint32_t bytes = what < 2 ? parts * (D / 2) : parts * U * 2;
		const int src0 = what < 2 ? what * cb : 2 * cb + (what - 2) * sb;
		const int dst0 = what < 2 ? what * L::CODES : 2 * L::CODES + (what - 2) * L::SCALES;
		const int row_bytes = what < 2 ? D / 2 : U * 2;
		int it = 0;
		while (left > 0)
		{
			const int n = min(left, s.tiles - tile), hk = seg / groups;
			const int* table = a.table + (size_t)s.r * a.table_stride;
			int ids = -1, base = -1; // 32 entries of the table from page `base`
			for (int t = tile; t < tile + n; ++t, ++it)
			{
				const int stage = it % STAGES;
				if (it >= STAGES && !*abort_ && !kv4_wait(&empty[stage], ((it / STAGES) - 1) & 1, ws.err, DEVERR_WAIT_EMPTY))
					*abort_ = 1;
				__syncwarp();
				const bool stop = __shfl_sync(0xffffffffu, *abort_, 0) != 0; // one answer for the warp
				const int key0 = (s.tile0 + t) * TILE, page0 = key0 >> a.page_shift;
				if (base < 0 || page0 + n_parts > base + 32)
				{
					base = page0;
					ids = base + lane < a.max_blocks ? table[base + lane] : -1;
				}
				const int k0 = key0 + part * parts; // this lane's part: its first key
				const int id = __shfl_sync(0xffffffffu, ids, page0 - base + (part < n_parts ? part : 0));
				const bool get = !stop && part < n_parts && id >= 0 && id < a.n_pages && k0 <= s.last && k0 + parts > s.first;
				const unsigned got = __ballot_sync(0xffffffffu, get);
				if (lane == 0)
				{
					int mask = got ? 15 : 0; // one part: all or nothing
					if (n_parts > 1)
					{
						mask = 0;
						for (int p = 0; p < n_parts; ++p)
							if (got >> (4 * p) & 1) mask |= (parts == 32 ? 3 : 1) << (p * (parts / 16));
					}
					loaded[stage] = mask;
					mbar_arrive_expect_tx(&full[stage], __popc(got) / 4 * 2 * (uint32_t)(parts * (D / 2) + parts * U * 2));
				}
				__syncwarp();
				if (get)
				{
					const int off = k0 & (a.page - 1);
					bulk_g2s(smem + stage * L::STAGE + dst0 + part * parts * row_bytes,
					         a.pages + ((size_t)id * a.n_kv + hk) * kv4_chunk_bytes(a.page, D) + src0 + off * row_bytes, bytes,
					         &full[stage]);
				}
			}
			next_piece(n);
		}
		// after a wait that ran out nobody may have waited for the copies in flight: not to leave before they landed
		if (*abort_)
			for (int i = max(0, it - STAGES); i < it; ++i)
				kv4_wait(&full[i % STAGES], (i / STAGES) & 1, nullptr, 0);
		return;
	}

	// ---- the computing warps ----
	const int c4 = lane & 3, i8 = lane >> 2;
	// K: this lane's two rows of the products, keys ka and ka + 8 of the warp's 16; V: keys c4 + 4 kk
	const int ka = warp * 16 + (i8 >> 1) + 4 * (i8 & 1);
	const int k_off = ka * (D / 2) + 16 * ((ka * D / 256) & (U - 1)) + 4 * c4;
	int v_off[2];
#pragma unroll
	for (int kk = 0; kk < 2; ++kk)
	{
		const int key = warp * 16 + c4 + 4 * kk;
		v_off[kk] = key * (D / 2) + 16 * (((i8 >> 2) * J) ^ ((key * D / 256) & (U - 1))) + 4 * (i8 & 3);
	}
	// scores in base 2 (with a soft-cap: its argument, and what multiplies its value)
	const float scale2 = a.softcap > 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
	const float softcap2 = a.softcap * 1.4426950408889634f;
	const Masks mk;
	int it = 0;
	while (left > 0)
	{
		const int n = min(left, s.tiles - tile), hk = seg / groups;
		s.row0 = (seg - hk * groups) * ROWS;

		// q's rows as operands: column i8 of row tile r is row s.row0 + 8 r + i8
		float mult[R][2];              // what turns a product into a base-2 score
		int at[R][2];                  // positions of columns 2 c4 and 2 c4 + 1 (-1: no row)
		float held[R][2], l[R][2];     // P_SCALE - held score, sum of the weights
		int all_from = 0, all_to = INT_MAX; // keys that every row sees
#pragma unroll
		for (int r = 0; r < R; ++r)
		{
			const int row = s.row0 + 8 * r + i8;
			const bool real = row < s.rows;
			const float* qp = nullptr;
			if (real)
			{
				const int t = row / a.group;
				qp = a.q + (size_t)(s.x.q0 + t) * a.q_stride + (size_t)(hk * a.group + row - t * a.group) * D + 8 * c4;
			}
			float v[U][8], top = 0.0f;
#pragma unroll
			for (int g = 0; g < U; ++g)
			{
				const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				const float4 x = real ? *reinterpret_cast<const float4*>(qp + 32 * g) : z;
				const float4 y = real ? *reinterpret_cast<const float4*>(qp + 32 * g + 4) : z;
				v[g][0] = x.x, v[g][1] = x.y, v[g][2] = x.z, v[g][3] = x.w;
				v[g][4] = y.x, v[g][5] = y.y, v[g][6] = y.z, v[g][7] = y.w;
#pragma unroll
				for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[g][e]));
			}
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
			// the power of two that brings the row's largest value to [2^14, 2^15)
			const int ex = top > 0.0f ? max(-100, min(100, ilogbf(top))) : 0;
			const float f = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
#pragma unroll
			for (int g = 0; g < U; ++g)
#pragma unroll
				for (int h = 0; h < 2; ++h)
				{
					if ((g & (CW - 1)) != warp) continue;
					uint32_t b[4]; // high halves of values 4h, 4h+1 | 4h+2, 4h+3, low halves
					split2(v[g][4 * h] * f, v[g][4 * h + 1] * f, b[0], b[2]);
					split2(v[g][4 * h + 2] * f, v[g][4 * h + 3] * f, b[1], b[3]);
					qsm[((2 * g + h) * R + r) * 32 + lane] = make_uint4(b[0], b[1], b[2], b[3]);
				}
#pragma unroll
			for (int e = 0; e < 2; ++e)
			{
				const int from = (2 * c4 + e) * 4;
				mult[r][e] = scale2 / __shfl_sync(0xffffffffu, f, from);
				const int row2 = s.row0 + 8 * r + 2 * c4 + e;
				at[r][e] = row2 < s.rows ? s.x.pos0 + row2 / a.group : -1;
				held[r][e] = NONE;
				l[r][e] = 0.0f;
				if (row2 < s.rows)
				{
					all_from = max(all_from, kv4_first_key(a, at[r][e]));
					all_to = min(all_to, min(at[r][e], s.x.keys - 1));
				}
			}
		}
#pragma unroll
		for (int o = 1; o < 4; o <<= 1)
		{
			all_from = max(all_from, __shfl_xor_sync(0xffffffffu, all_from, o));
			all_to = min(all_to, __shfl_xor_sync(0xffffffffu, all_to, o));
		}
		named_sync(1, CW * 32);

		float o[J * 4][R][4];
#pragma unroll
		for (int x = 0; x < J * 4; ++x)
#pragma unroll
			for (int r = 0; r < R; ++r)
#pragma unroll
				for (int e = 0; e < 4; ++e) o[x][r][e] = 0.0f;
		bool bad = false; // a V scale was no number

		for (int t = tile; t < tile + n; ++t, ++it)
		{
			const int stage = it % STAGES;
			const bool came = !*abort_ && kv4_wait(&full[stage], (it / STAGES) & 1, ws.err, DEVERR_WAIT_FULL);
			if (!came) *abort_ = 1;
			const unsigned char* st = smem + stage * L::STAGE;
			const int key0 = (s.tile0 + t) * TILE + warp * 16;
			// (one answer for the warp, whose lanes work together below: after a wait that ran out they might see different ones)
			if (__all_sync(0xffffffffu, came && (loaded[stage] >> warp & 1)))
			{
				// ---- scores of 16 keys ----
				float sc[R][4];
#pragma unroll
				for (int r = 0; r < R; ++r)
#pragma unroll
					for (int e = 0; e < 4; ++e) sc[r][e] = 0.0f;
				float ks[2][U];
				load_scales<U>(ks[0], st + 2 * L::CODES + ka * (2 * U));
				load_scales<U>(ks[1], st + 2 * L::CODES + (ka + 8) * (2 * U));
#pragma unroll
				for (int g = 0; g < U; ++g)
				{
					const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + (k_off ^ (16 * g)));
					const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + (k_off ^ (16 * g)) + 8 * (D / 2));
					uint32_t k0[4], k1[4]; // the codes of both keys, pair by pair
#pragma unroll
					for (int x = 0; x < 4; ++x) k0[x] = half2_bits(codes2(mk, w0, x)), k1[x] = half2_bits(codes2(mk, w1, x));
#pragma unroll
					for (int r = 0; r < R; ++r)
					{
						float d[4];
						const uint4 b = qsm[(2 * g * R + r) * 32 + lane], e = qsm[((2 * g + 1) * R + r) * 32 + lane];
						mma16816_first(d, k0[0], k1[0], k0[1], k1[1], b.x, b.y);
						mma16816(d, k0[0], k1[0], k0[1], k1[1], b.z, b.w);
						mma16816(d, k0[2], k1[2], k0[3], k1[3], e.x, e.y);
						mma16816(d, k0[2], k1[2], k0[3], k1[3], e.z, e.w);
						sc[r][0] = fmaf(d[0], ks[0][g], sc[r][0]);
						sc[r][1] = fmaf(d[1], ks[0][g], sc[r][1]);
						sc[r][2] = fmaf(d[2], ks[1][g], sc[r][2]);
						sc[r][3] = fmaf(d[3], ks[1][g], sc[r][3]);
					}
				}
				// ---- weights ----
				const bool edge = key0 < all_from || key0 + 15 > all_to;
				uint32_t ph[R][2], pl[R][2]; // [keys 0-7 | 8-15], transposed: the second product's operand
				if (a.softcap > 0.0f)
				{
#pragma unroll
					for (int r = 0; r < R; ++r)
#pragma unroll
						for (int e = 0; e < 4; ++e) sc[r][e] = tanhf(sc[r][e] * mult[r][e & 1]) * softcap2;
				}
				else
				{
#pragma unroll
					for (int r = 0; r < R; ++r)
#pragma unroll
						for (int e = 0; e < 4; ++e) sc[r][e] *= mult[r][e & 1];
				}
				if (edge)
				{
					const int kx = key0 + (ka & 15), end = s.x.keys;
#pragma unroll
					for (int r = 0; r < R; ++r)
#pragma unroll
						for (int e = 0; e < 4; ++e)
						{
							const int k = kx + (e & 2 ? 8 : 0), pos = at[r][e & 1];
							if (k > pos || k >= end || (a.window > 0 && pos - k >= a.window)) sc[r][e] = -CUDART_INF_F;
						}
				}
#pragma unroll
				for (int r = 0; r < R; ++r)
				{
					const float t0 = fmaxf(sc[r][0], sc[r][2]) + held[r][0], t1 = fmaxf(sc[r][1], sc[r][3]) + held[r][1];
					if (__any_sync(0xffffffffu, fmaxf(t0, t1) > P_TOP))
					{
#pragma unroll
						for (int e = 0; e < 2; ++e)
						{
							float top = fmaxf(sc[r][e], sc[r][e + 2]);
#pragma unroll
							for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
							if (top + held[r][e] > P_TOP)
							{
								const float alpha = ex2(P_SCALE - top - held[r][e]);
								held[r][e] = P_SCALE - top;
								l[r][e] *= alpha;
#pragma unroll
								for (int x = 0; x < J * 4; ++x)
								{
									o[x][r][e] *= alpha;
									o[x][r][e + 2] *= alpha;
								}
							}
						}
					}
#pragma unroll
					for (int e = 0; e < 4; ++e)
					{
						sc[r][e] = ex2(sc[r][e] + held[r][e & 1]);
						l[r][e & 1] += sc[r][e];
					}
#pragma unroll
					for (int h = 0; h < 2; ++h)
					{
						uint32_t hi, lo;
						split2(sc[r][2 * h], sc[r][2 * h + 1], hi, lo);
						ph[r][h] = transpose8(hi);
						pl[r][h] = transpose8(lo);
					}
				}
				// ---- values: keys c4 + 4 kk of the warp's 16, J words of codes each ----
				float vs[4][J];
#pragma unroll
				for (int kk = 0; kk < 4; ++kk)
					load_scales<J>(vs[kk], st + 2 * L::CODES + L::SCALES + ((warp * 16 + c4 + 4 * kk) * U + (i8 >> 2) * J) * 2);
				if (edge)
#pragma unroll
					for (int kk = 0; kk < 4; ++kk)
						if (key0 + c4 + 4 * kk < s.first || key0 + c4 + 4 * kk > s.last) // whatever was there
#pragma unroll
							for (int j = 0; j < J; ++j) vs[kk][j] = 0.0f;
				__half2 s2[J][2]; // the scales of key pairs (0, 1) and (2, 3)
				__half2 odd = __float2half2_rn(0.0f);
#pragma unroll
				for (int j = 0; j < J; ++j)
#pragma unroll
					for (int pr = 0; pr < 2; ++pr)
					{
						s2[j][pr] = __floats2half2_rn(vs[2 * pr][j], vs[2 * pr + 1][j]);
						odd = __hfma2(s2[j][pr], __float2half2_rn(0.0f), odd); // no number where a scale is none (or no 16-bit one)
					}
				if (__any_sync(0xffffffffu, __hisnan(__low2half(odd)) || __hisnan(__high2half(odd))))
				{
					// goes in as a number: zero weights must stay zero for the rows that do not see its key. (Finite
					// scales are within these bounds.)
					bad = true;
#pragma unroll
					for (int j = 0; j < J; ++j)
#pragma unroll
						for (int pr = 0; pr < 2; ++pr)
							s2[j][pr] = __hmax2(__hmin2(s2[j][pr], __float2half2_rn(KV4_SCALE_MAX)), __float2half2_rn(-KV4_SCALE_MAX));
				}
#pragma unroll
				for (int j = 0; j < J; ++j)
				{
					uint32_t lo[2], hi[2];
#pragma unroll
					for (int pr = 0; pr < 2; ++pr)
					{
						const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + L::CODES + (v_off[0] ^ (16 * j)) + pr * 8 * (D / 2));
						const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + L::CODES + (v_off[1] ^ (16 * j)) + pr * 8 * (D / 2));
						lo[pr] = __byte_perm(w0, w1, 0x5410);
						hi[pr] = __byte_perm(w0, w1, 0x7632);
					}
#pragma unroll
					for (int x = 0; x < 4; ++x)
					{
						const auto widen = [&](uint32_t w, int pr) { return half2_bits(__hmul2(codes2(mk, w, x), s2[j][pr])); };
						const uint32_t a0 = widen(lo[0], 0), a1 = widen(hi[0], 0), a2 = widen(lo[1], 1), a3 = widen(hi[1], 1);
#pragma unroll
						for (int r = 0; r < R; ++r)
						{
							mma16816(o[j * 4 + x][r], a0, a1, a2, a3, ph[r][0], ph[r][1]);
							mma16816(o[j * 4 + x][r], a0, a1, a2, a3, pl[r][0], pl[r][1]);
						}
					}
				}
			}
			__syncwarp();
			if (lane == 0) mbar_arrive(&empty[stage]);
		}

		// ---- the piece's end: the four warps' states joined ----
		float m[R][2];
#pragma unroll
		for (int r = 0; r < R; ++r)
#pragma unroll
			for (int e = 0; e < 2; ++e)
			{
#pragma unroll
				for (int w = 4; w < 32; w <<= 1) l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], w);
				m[r][e] = held[r][e] == NONE ? -CUDART_INF_F : P_SCALE - held[r][e];
				if (i8 == 0) ml[warp * ROWS + 8 * r + 2 * c4 + e] = make_float2(m[r][e], l[r][e]);
			}
		const bool any_bad = named_sync_or(1, CW * 32, bad);
#pragma unroll
		for (int r = 0; r < R; ++r)
#pragma unroll
			for (int e = 0; e < 2; ++e)
			{
				const int col = 8 * r + 2 * c4 + e;
				float top = ml[col].x;
#pragma unroll
				for (int w = 1; w < CW; ++w) top = fmaxf(top, ml[w * ROWS + col].x);
				const float f = m[r][e] == top ? 1.0f : ex2(m[r][e] - top);
				float* dst = red + (warp * ROWS + col) * L::RED_ROW + 32 * ((i8 >> 2) * J) + 8 * (i8 & 3);
#pragma unroll
				for (int j = 0; j < J; ++j)
				{
					float4 y[2];
					y[0] = make_float4(o[4 * j][r][e] * f, o[4 * j][r][e + 2] * f, o[4 * j + 1][r][e] * f, o[4 * j + 1][r][e + 2] * f);
					y[1] = make_float4(o[4 * j + 2][r][e] * f, o[4 * j + 2][r][e + 2] * f, o[4 * j + 3][r][e] * f,
					                   o[4 * j + 3][r][e + 2] * f);
					reinterpret_cast<float4*>(dst + 32 * j)[0] = y[0];
					reinterpret_cast<float4*>(dst + 32 * j)[1] = y[1];
				}
			}
		// (the weights of a row, for the threads that finish it below)
		constexpr int QUADS = D / 4, MINE = ROWS * QUADS / (CW * 32);
		float top[MINE], sum[MINE];
#pragma unroll
		for (int x = 0; x < MINE; ++x)
		{
			const int row = (tid + x * CW * 32) / QUADS;
			top[x] = ml[row].x;
#pragma unroll
			for (int w = 1; w < CW; ++w) top[x] = fmaxf(top[x], ml[w * ROWS + row].x);
			sum[x] = 0.0f;
#pragma unroll
			for (int w = 0; w < CW; ++w)
			{
				const float2 y = ml[w * ROWS + row];
				sum[x] = fmaf(y.y, y.x == top[x] ? 1.0f : ex2(y.x - top[x]), sum[x]);
			}
		}
		named_sync(1, CW * 32);
		const bool whole = tile == 0 && n == s.tiles;
		const int c_first = whole ? 0 : runs.owner(seg_at), c_last = whole ? 0 : runs.owner(seg_at + s.tiles - 1);
		// where CTA c's piece of this segment lies: behind its first, if the segment begins inside its run
		const auto slot = [&](int c) {
			return ws.parts + (size_t)(2 * c + (c == c_first && runs.begin(c) < seg_at)) * L::PART;
		};
#pragma unroll
		for (int x = 0; x < MINE; ++x)
		{
			const int item = tid + x * CW * 32, row = item / QUADS, d = item % QUADS * 4;
			float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
			for (int w = 0; w < CW; ++w)
			{
				const float4 z = *reinterpret_cast<const float4*>(red + (w * ROWS + row) * L::RED_ROW + d);
				y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
			}
			const int rr = s.row0 + row;
			if (any_bad && rr < s.rows)
			{
				// a row that sees a value that is no number has none in the group
				const int pos = s.x.pos0 + rr / a.group;
				const int from = max(kv4_first_key(a, pos), (s.tile0 + tile) * TILE);
				const int to = min(min(pos, s.x.keys - 1), (s.tile0 + tile + n) * TILE - 1);
				for (int k = from; k <= to; ++k)
				{
					const int id = a.table[(size_t)s.r * a.table_stride + (k >> a.page_shift)];
					if (id < 0 || id >= a.n_pages) continue;
					const uint8_t* chunk = a.pages + ((size_t)id * a.n_kv + hk) * kv4_chunk_bytes(a.page, D);
					const uint16_t* vs = reinterpret_cast<const uint16_t*>(chunk + 2 * kv4_codes_bytes(a.page, D) +
					                                                       kv4_scales_bytes(a.page, D));
					const float f = bf16_bits_to_float(vs[(k & (a.page - 1)) * U + d / KV4_GROUP]);
					if (!(fabsf(f) <= KV4_SCALE_MAX)) y.x = y.y = y.z = y.w = CUDART_NAN_F;
				}
			}
			if (whole)
			{
				if (rr < s.rows)
				{
					const float inv = sum[x] == 0.0f ? 0.0f : 1.0f / sum[x];
					const int tk = rr / a.group;
					*reinterpret_cast<float4*>(a.out + (size_t)(s.x.q0 + tk) * a.out_stride +
					                           (size_t)(hk * a.group + rr - tk * a.group) * D + d) =
						make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
				}
			}
			else
			{
				float* p = slot(blockIdx.x);
				*reinterpret_cast<float4*>(p + row * D + d) = y;
				if (d == 0) *reinterpret_cast<float2*>(p + ROWS * D + 2 * row) = make_float2(top[x], sum[x]);
			}
		}
		if (!whole)
		{
			named_sync(1, CW * 32);
			if (tid == 0)
			{
				// (releases what the barrier has gathered, acquires what the others released)
				int was;
				asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(was) : "l"(&ws.counters[c_first]) : "memory");
				*last_piece = was == c_last - c_first;
				if (*last_piece) ws.counters[c_first] = 0; // ready for the next call
			}
			named_sync(1, CW * 32);
			if (*last_piece)
			{
				// the last piece of the segment: all of them joined, in order (the largest maximum first: then the
				// parts' loads wait for nothing but each other's places)
				float mx[MINE], w[MINE];
				float4 y[MINE];
#pragma unroll
				for (int x = 0; x < MINE; ++x) mx[x] = -CUDART_INF_F, w[x] = 0.0f, y[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
				for (int c = c_first; c <= c_last; ++c)
#pragma unroll
					for (int x = 0; x < MINE; ++x)
						mx[x] = fmaxf(mx[x], __ldcg(slot(c) + ROWS * D + 2 * ((tid + x * CW * 32) / QUADS)));
#pragma unroll(MINE <= 2 ? 8 : 2)
				for (int c = c_first; c <= c_last; ++c)
				{
					const float* p = slot(c);
#pragma unroll
					for (int x = 0; x < MINE; ++x)
					{
						const int item = tid + x * CW * 32, row = item / QUADS, d = item % QUADS * 4;
						const float2 z = __ldcg(reinterpret_cast<const float2*>(p + ROWS * D + 2 * row));
						const float4 u = __ldcg(reinterpret_cast<const float4*>(p + row * D + d));
						const float f = z.x == mx[x] ? 1.0f : ex2(z.x - mx[x]);
						w[x] = fmaf(z.y, f, w[x]);
						y[x].x = fmaf(u.x, f, y[x].x), y[x].y = fmaf(u.y, f, y[x].y);
						y[x].z = fmaf(u.z, f, y[x].z), y[x].w = fmaf(u.w, f, y[x].w);
					}
				}
#pragma unroll
				for (int x = 0; x < MINE; ++x)
				{
					const int item = tid + x * CW * 32, rr = s.row0 + item / QUADS, d = item % QUADS * 4;
					if (rr >= s.rows) continue;
					const float inv = w[x] == 0.0f ? 0.0f : 1.0f / w[x];
					const int tk = rr / a.group;
					*reinterpret_cast<float4*>(a.out + (size_t)(s.x.q0 + tk) * a.out_stride +
					                           (size_t)(hk * a.group + rr - tk * a.group) * D + d) =
						make_float4(y[x].x * inv, y[x].y * inv, y[x].z * inv, y[x].w * inv);
				}
			}
		}
		next_piece(n);
	}
}

constexpr int MAX_SMS = 192;
// the counters' place is the same for every variant: one workspace serves them all in turn
constexpr size_t WS_PARTS = 256 + 4096;

template <int D, int R>
constexpr size_t ws_bytes(int sms)
{
	const size_t ctas = (size_t)sms * Shape<D, R>::CTAS;
	return (WS_PARTS + ctas * 2 * Shape<D, R>::PART * 4 + 255) / 256 * 256;
}
size_t ws_bytes(int D) // enough for every variant of the head_dim on any device of this kind
{
	static_assert(ws_bytes<64, 4>(1) >= ws_bytes<64, 3>(1) && ws_bytes<64, 4>(1) >= ws_bytes<64, 2>(1) && ws_bytes<64, 4>(1) >= ws_bytes<64, 1>(1) &&
	                  ws_bytes<128, 2>(1) >= ws_bytes<128, 1>(1),
	              "the largest variant");
	return D == 64 ? ws_bytes<64, 4>(MAX_SMS) : D == 128 ? ws_bytes<128, 2>(MAX_SMS) : ws_bytes<256, 1>(MAX_SMS);
}

int num_sms()
{
	static int known[64] = {};
	int dev = 0;
	if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
	if (known[dev] == 0 && cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
		return 0;
	return known[dev];
}

template <int D, int R>
int launch_decode4(const Kv4Args& a, void* workspace, cudaStream_t st)
{
	using L = Shape<D, R>;
	static bool configured[64] = {};
	int dev = 0;
	cudaGetDevice(&dev);
	if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
	auto kernel = kv4_decode_kernel<D, R>;
	if (!configured[dev])
	{
		const cudaError_t ce = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
		if (ce != cudaSuccess) return (int)ce;
		configured[dev] = true;
	}
	const int ctas = num_sms() * L::CTAS;
	if (ctas == 0 || ctas > MAX_SMS * L::CTAS) return (int)cudaErrorInvalidDevice;
	unsigned char* w = static_cast<unsigned char*>(workspace);
	const Ws ws{reinterpret_cast<int*>(w), reinterpret_cast<int*>(w + 256),
	            reinterpret_cast<float*>(w + WS_PARTS)};
	kernel<<<ctas, THREADS, L::SMEM, st>>>(a, ws);
	note_launches(1);
	return (int)cudaGetLastError();
}

// The most key tiles that a call can have, by what its tables can hold.
long long most_tiles(const nncu_kv4_attn* a)
{
	const long long span = (long long)a->max_blocks * a->pool.page_size, seen = (long long)a->window + a->max_new;
	return (a->window > 0 && seen < span ? seen : span) / TILE * a->n_req * a->pool.n_kv;
}
int few_rows_of(const nncu_kv4_attn* a)
{
	return most_tiles(a) < FEW_TILES ? 2 * few_rows(a->pool.head_dim) : few_rows(a->pool.head_dim);
}

int refuse(const char* msg) { return set_error(NNCU_ERR_INVALID_ARGUMENT, msg); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What an attention call and its workspace both need to hold.
int check_shape(const nncu_kv4_attn* a, bool need_pages)
{
	if (!a) return refuse("kv4 attention: NULL argument");
	const int rc = kv4_check_pool(&a->pool, "kv4 attention", need_pages);
	if (rc != NNCU_OK) return rc;
	if (a->n_req < 0 || a->n_tok < 0 || a->max_new < 0 || a->max_blocks < 0 || a->window < 0)
		return refuse("kv4 attention: negative n_req, n_tok, max_new, max_blocks or window");
	if (a->n_head <= 0 || a->n_head % a->pool.n_kv) return refuse("kv4 attention: n_head must be a multiple of n_kv");
	if ((long long)a->max_blocks * a->pool.page_size > INT32_MAX - 256)
		return refuse("kv4 attention: max_blocks x page_size passes 2^31");
	// rows, and the tensor-core kernel's CTAs, are numbered with 32 bits
	const long long group = a->n_head / a->pool.n_kv, rows = group * a->n_tok;
	if (rows > INT32_MAX / 2 || group * a->max_new > INT32_MAX / 2 ||
	    (rows / 128 + a->n_req + 1024) * a->pool.n_kv > INT32_MAX)
		return refuse("kv4 attention: n_tok, n_req and heads together pass 2^31");
	return NNCU_OK;
}

} // namespace
} // namespace nncu

using namespace nncu;

extern "C" int nncu_kv4_workspace_bytes(const nncu_kv4_attn* a, size_t* bytes)
{
	const int rc = check_shape(a, false);
	if (rc != NNCU_OK) return rc;
	if (!bytes) return refuse("kv4 workspace: NULL argument");
	*bytes = ws_bytes(a->pool.head_dim);
	const long long group = a->n_head / a->pool.n_kv;
	if (group * a->max_new > few_rows_of(a))
		*bytes = kv4_prompt_ws_end(a->pool.head_dim, *bytes, a->n_req, group * a->n_tok, a->pool.n_kv);
	return NNCU_OK;
}

extern "C" int nncu_kv4_check(const nncu_kv4_attn* a, void* stream)
{
	if (!a || !a->workspace || a->workspace_bytes < 256) return refuse("kv4 check: NULL argument or workspace");
	const auto st = static_cast<cudaStream_t>(stream);
	int err = 0;
	cudaError_t ce = cudaMemcpyAsync(&err, a->workspace, sizeof err, cudaMemcpyDeviceToHost, st);
	if (ce == cudaSuccess) ce = cudaStreamSynchronize(st);
	if (ce != cudaSuccess) return set_cuda_error((int)ce, "kv4 check");
	if (err == 0) return NNCU_OK;
	ce = cudaMemsetAsync(a->workspace, 0, a->workspace_bytes, st);
	if (ce == cudaSuccess) ce = cudaStreamSynchronize(st);
	if (ce != cudaSuccess) return set_cuda_error((int)ce, "kv4 check");
	return set_error(NNCU_ERR_TIMEOUT, "kv4 attention: a kernel's bounded wait ran out; its outputs are void");
}

extern "C" int nncu_kv4_attention_dev(const nncu_kv4_attn* p, void* stream)
{
	int rc = check_shape(p, true);
	if (rc != NNCU_OK) return rc;
	if (p->n_req == 0 || p->n_tok == 0 || p->max_new == 0) return NNCU_OK;
	if (!p->block_table || !p->seq_len || !p->q_start || !p->q || !p->out)
		return refuse("kv4 attention: NULL array");
	if (p->max_blocks == 0 || p->table_stride < (size_t)p->max_blocks)
		return refuse("kv4 attention: table rows shorter than max_blocks");
	if (!aligned16(p->q) || !aligned16(p->out) || p->q_stride % 4 || p->out_stride % 4)
		return refuse("kv4 attention: q and out rows must be 16-byte aligned");
	const size_t row = (size_t)p->n_head * p->pool.head_dim;
	if (p->n_tok > 1 && (p->q_stride < row || p->out_stride < row))
		return refuse("kv4 attention: strides shorter than a row");
	if (!(p->softcap >= 0.0f) || std::isinf(p->softcap) || !std::isfinite(p->scale))
		return refuse("kv4 attention: bad scale or softcap");
	size_t need = 0;
	rc = nncu_kv4_workspace_bytes(p, &need);
	if (rc != NNCU_OK) return rc;
	if (!p->workspace || !aligned16(p->workspace) || p->workspace_bytes < need)
	{
		char msg[120];
		snprintf(msg, sizeof msg, "kv4 attention: a 16-byte aligned workspace of %zu bytes is needed", need);
		return refuse(msg);
	}
	int shift = 0;
	while ((1 << shift) < p->pool.page_size) ++shift;
	const Kv4Args a{static_cast<const uint8_t*>(p->pool.pages), p->pool.n_pages, p->pool.page_size, shift,
	                p->pool.n_kv, p->pool.head_dim, p->n_req, p->n_tok, p->n_head, p->n_head / p->pool.n_kv,
	                p->max_new, p->max_blocks, p->window, few_rows_of(p), p->scale, p->softcap, p->block_table, p->table_stride,
	                p->seq_len, p->q_start, p->q, p->q_stride, p->out, p->out_stride};
	const auto st = static_cast<cudaStream_t>(stream);
	const long long rows = (long long)a.group * p->max_new;
	// (a call that may have prompts still decodes the requests with few rows here)
	const long long few = rows < a.few_rows ? rows : a.few_rows, tiles8 = (few + 7) / 8, tiles = most_tiles(p);
	int e;
	if (a.D == 256)
		e = launch_decode4<256, 1>(a, p->workspace, st);
	else if (a.D == 128)
		// (three row tiles: 93 us one by one, 99 as two and one)
		e = tiles < MANY_TILES || (tiles8 & 1 && tiles8 < 4) ? launch_decode4<128, 1>(a, p->workspace, st)
		                                                     : launch_decode4<128, 2>(a, p->workspace, st);
	else
		e = tiles < MANY_TILES || tiles8 == 1 ? launch_decode4<64, 1>(a, p->workspace, st)
		    : tiles8 == 2                     ? launch_decode4<64, 2>(a, p->workspace, st)
		    : tiles8 == 3                     ? launch_decode4<64, 3>(a, p->workspace, st)
		                                      : launch_decode4<64, 4>(a, p->workspace, st);
	if (!e && rows > a.few_rows) e = launch_kv4_prompt(a, p->workspace, ws_bytes(a.D), a.few_rows, stream);
	return e ? set_cuda_error(e, "kv4 attention launch") : NNCU_OK;
}
