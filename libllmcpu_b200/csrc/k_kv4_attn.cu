// k_kv4_attn.cu -- attention of packed requests over the paged 4-bit cache
// (nncu_kv4_attention_dev): decode, verify and prompt.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstdio>

#include "kv4.cuh"

namespace nncu
{
namespace
{

constexpr int SIMPLE_WARPS = 4;

// One CTA per (token, query head); the warps take keys in turn, every lane
// D / 32 neighbouring values, and join their softmax states at the end.
template <int D>
__global__ void __launch_bounds__(SIMPLE_WARPS * 32) kv4_simple_kernel(const Kv4Args a)
{
	constexpr int E = D / 32, U = D / KV4_GROUP;
	__shared__ float so[SIMPLE_WARPS][D], sm[SIMPLE_WARPS], sl[SIMPLE_WARPS];
	const int t = blockIdx.x, h = blockIdx.y, hk = h / a.group;
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	// the request of this token (the last whose first token is not past it)
	int lo = 0, hi = a.n_req - 1;
	while (lo < hi)
	{
		const int mid = (lo + hi + 1) >> 1;
		if (a.q_start[mid] <= t)
			lo = mid;
		else
			hi = mid - 1;
	}
	const Kv4Request x = kv4_request(a, lo);
	if (t < x.q0 || t - x.q0 >= x.n_new) return;
	const int pos = x.pos0 + t - x.q0;
	const int last = min(pos, x.keys - 1), first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
	float q[E], o[E], m = -CUDART_INF_F, l = 0.0f;
	const float* qp = a.q + (size_t)t * a.q_stride + (size_t)h * D + lane * E;
#pragma unroll
	for (int e = 0; e < E; ++e) q[e] = qp[e], o[e] = 0.0f;
	const int v0 = lane * E, g = v0 / KV4_GROUP;
	const int cb = kv4_codes_bytes(a.page, D), sb = kv4_scales_bytes(a.page, D);
	for (int k = first + warp; k <= last; k += SIMPLE_WARPS)
	{
		const int pg = a.table[(size_t)lo * a.table_stride + (k >> a.page_shift)];
		if (pg < 0 || pg >= a.n_pages) continue;
		const int off = k & (a.page - 1);
		const uint8_t* chunk = a.pages + ((size_t)pg * a.n_kv + hk) * kv4_chunk_bytes(a.page, D);
		const uint8_t* row = chunk + off * (D / 2) + 16 * kv4_unit(off, g, D) + (v0 % KV4_GROUP) / 8 * 4;
		const uint16_t* sc = reinterpret_cast<const uint16_t*>(chunk + 2 * cb) + off * U + g;
		const uint32_t kw = *reinterpret_cast<const uint32_t*>(row), vw = *reinterpret_cast<const uint32_t*>(row + cb);
		const float ks = bf16_bits_to_float(sc[0]), vs = bf16_bits_to_float(sc[sb / 2]);
		float s = 0.0f;
#pragma unroll
		for (int e = 0; e < E; ++e)
			s = fmaf(q[e], ks * (float)((int)((kw >> (4 * kv4_nibble((v0 + e) & 7))) & 15u) - 8), s);
		s = warp_sum(s) * a.scale;
		if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
		const float mn = fmaxf(m, s);
		const float c = mn == -CUDART_INF_F ? 0.0f : expf(m - mn), p = mn == -CUDART_INF_F ? 0.0f : expf(s - mn);
		l = l * c + p;
#pragma unroll
		for (int e = 0; e < E; ++e)
			o[e] = o[e] * c + p * (vs * (float)((int)((vw >> (4 * kv4_nibble((v0 + e) & 7))) & 15u) - 8));
		m = mn;
	}
#pragma unroll
	for (int e = 0; e < E; ++e) so[warp][v0 + e] = o[e];
	if (lane == 0) sm[warp] = m, sl[warp] = l;
	__syncthreads();
	float mm = -CUDART_INF_F, ll = 0.0f;
	for (int w = 0; w < SIMPLE_WARPS; ++w) mm = fmaxf(mm, sm[w]);
	float f[SIMPLE_WARPS];
	for (int w = 0; w < SIMPLE_WARPS; ++w)
	{
		f[w] = sm[w] == -CUDART_INF_F ? 0.0f : expf(sm[w] - mm);
		ll += f[w] * sl[w];
	}
	for (int d = threadIdx.x; d < D; d += blockDim.x)
	{
		float y = 0.0f;
		for (int w = 0; w < SIMPLE_WARPS; ++w)
			if (f[w] != 0.0f) y += f[w] * so[w][d];
		a.out[(size_t)t * a.out_stride + (size_t)h * D + d] = ll != 0.0f ? y / ll : 0.0f;
	}
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
	if ((long long)a->max_blocks * a->pool.page_size > INT32_MAX)
		return refuse("kv4 attention: max_blocks x page_size passes 2^31");
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
	*bytes = 256;
	return NNCU_OK;
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
	if (!(p->softcap >= 0.0f) || !(p->scale == p->scale)) return refuse("kv4 attention: bad scale or softcap");
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
	                p->max_new, p->max_blocks, p->window, p->scale, p->softcap, p->block_table, p->table_stride,
	                p->seq_len, p->q_start, p->q, p->q_stride, p->out, p->out_stride};
	const auto st = static_cast<cudaStream_t>(stream);
	const dim3 grid((unsigned)p->n_tok, (unsigned)p->n_head);
	switch (p->pool.head_dim)
	{
	case 64: kv4_simple_kernel<64><<<grid, SIMPLE_WARPS * 32, 0, st>>>(a); break;
	case 128: kv4_simple_kernel<128><<<grid, SIMPLE_WARPS * 32, 0, st>>>(a); break;
	default: kv4_simple_kernel<256><<<grid, SIMPLE_WARPS * 32, 0, st>>>(a); break;
	}
	note_launches(1);
	const int e = (int)cudaGetLastError();
	return e ? set_cuda_error(e, "kv4 attention launch") : NNCU_OK;
}
