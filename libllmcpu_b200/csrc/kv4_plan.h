// kv4_plan.h -- how the planning kernel of the prompts' attention cuts blocks
// of query rows into pieces (k_kv4_prompt.cu). Plain C++.
#pragma once

namespace nncu
{

constexpr int KV4_SHARES = 2 * 148; // pieces are about total / KV4_SHARES tiles long, and not under KV4_MIN_PIECE
constexpr int KV4_MIN_PIECE = 8;

// The most tiles of a piece, for `total` tiles of all blocks under each of
// n_kv KV heads. (A million tokens with many heads pass 2^31 tiles.)
constexpr int kv4_longest(long long total, int n_kv)
{
	const long long share = (total * n_kv + KV4_SHARES - 1) / KV4_SHARES;
	return share < KV4_MIN_PIECE ? KV4_MIN_PIECE : share > 0x7fffffff ? 0x7fffffff : (int)share;
}

} // namespace nncu
