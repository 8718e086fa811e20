// kv4.cuh -- the 4-bit paged cache's layout (nncu_kv4_pool, include/nncu.h) as
// the kernels see it: where a key's units and scales sit, and the codes of a
// 32-bit word.
#pragma once

#include <stdint.h>

#include "common.cuh"
#include "nncu.h"

namespace nncu
{

constexpr int KV4_GROUP = 32;              // values that share a scale
constexpr float KV4_SCALE_MIN = 0x1p-17f;  // below: an 11-bit product would not be exact in a 16-bit float
constexpr float KV4_SCALE_MAX = 0x1p11f;   // -8 times it is 2^14: well within one

// Bytes of one (page, KV head): K codes, V codes, K scales, V scales.
__host__ __device__ constexpr int kv4_codes_bytes(int page, int D) { return page * D / 2; }
__host__ __device__ constexpr int kv4_scales_bytes(int page, int D) { return page * (D / KV4_GROUP) * 2; }
__host__ __device__ constexpr size_t kv4_chunk_bytes(int page, int D)
{
	return 2 * (size_t)(kv4_codes_bytes(page, D) + kv4_scales_bytes(page, D));
}

// The unit (of 16 bytes, D / 32 a key) where group g of the key at offset
// `off` sits: swizzled by the key's 128-byte line, so that 8 keys' same group
// lies in 8 different bank quads of shared memory whatever the head_dim.
__host__ __device__ __forceinline__ int kv4_unit(int off, int g, int D)
{
	return g ^ ((off * (D / 2) / 128) & (D / KV4_GROUP - 1));
}

// Value `i` (0..7) of a word sits in this nibble: neighbours share a 16-bit
// lane pair (nibbles n and n + 4 are values 2n and 2n + 1), so masking a word
// gives two neighbouring values in the two halves of a register.
__host__ __device__ __forceinline__ int kv4_nibble(int i) { return (i >> 1) + 4 * (i & 1); }

__device__ __forceinline__ float bf16_bits_to_float(uint32_t b) { return __uint_as_float(b << 16); }

// The pool and the requests of one attention call, as the kernels get them.
struct Kv4Args
{
	const uint8_t* pages;
	int n_pages, page, page_shift, n_kv, D;
	int n_req, n_tok, n_head, group, max_new, max_blocks, window;
	int few_rows; // requests with more query rows a KV head are the tensor-memory kernel's
	float scale, softcap;
	const int* table;
	size_t table_stride;
	const int* seq_len;
	const int* q_start;
	const float* q;
	size_t q_stride;
	float* out;
	size_t out_stride;
};

// Wait for phase `parity` of `bar`, giving up after WAIT_LIMIT_NS (false, with
// `code` in the error word where there is one). The thread sleeps up to 1 ms
// at a time: these kernels have many warps waiting for one another, and short
// polls would take the issue slots of those that work.
__device__ __forceinline__ bool kv4_wait(uint64_t* bar, uint32_t parity, int* err, int code)
{
	const auto poll = [&]() {
		uint32_t ok;
		asm volatile("{\n\t.reg .pred p;\n\t"
		             "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
		             "selp.u32 %0, 1, 0, p;\n\t}"
		             : "=r"(ok)
		             : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
		             : "memory");
		return ok != 0;
	};
	if (poll()) return true;
	const uint64_t t0 = globaltimer_ns();
	do
		if (poll()) return true;
	while (globaltimer_ns() - t0 <= WAIT_LIMIT_NS);
	if (err) atomicCAS(err, 0, code);
	return false;
}

// The first key that a query at `pos` sees. (Written so that no position, below zero too, and no window overflow.)
__device__ __forceinline__ int kv4_first_key(const Kv4Args& a, int pos)
{
	return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
}

// One request's place in the packed tokens and its keys.
struct Kv4Request
{
	int q0, n_new, keys; // first token, tokens (within max_new and n_tok), keys in the cache
	int pos0;            // position of the first token
};
__device__ __forceinline__ Kv4Request kv4_request(const Kv4Args& a, int r)
{
	Kv4Request x;
	const int s = max(0, a.q_start[r]), e = a.q_start[r + 1];
	const int n = max(0, e - s);
	x.q0 = s;
	x.keys = max(0, min(a.seq_len[r], a.max_blocks << a.page_shift)); // (a length past its table row: the row's end)
	x.pos0 = x.keys - n;
	x.n_new = max(0, min(min(n, a.max_new), a.n_tok - s));
	return x;
}

// A pool's geometry (and, unless told otherwise, its pages) checked:
// NNCU_OK or the refusal (k_paged.cu).
int kv4_check_pool(const nncu_kv4_pool* p, const char* what, bool need_pages = true);

// The tensor-core kernel for requests with more than min_rows query rows
// (k_kv4_prompt.cu), its workspace from byte `at` of the call's; and where
// that ends for n_req requests with `rows` query rows a KV head together.
int launch_kv4_prompt(const Kv4Args& a, void* workspace, size_t at, int min_rows, void* stream);
size_t kv4_prompt_ws_end(int D, size_t at, int n_req, long long rows, int n_kv);

} // namespace nncu
