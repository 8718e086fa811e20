// i8_plan.h -- which kernel multiplies 8-bit rows, with what tile, split and
// stages (k_i8_linear.cu). Plain C++.
#pragma once

#include <algorithm>
#include <cmath>

namespace nncu
{

constexpr int I8_KB = 128;              // columns of a panel: one swizzled row
constexpr int I8_W_BYTES = 128 * I8_KB; // a panel's 128 channels
constexpr int I8_MAX_STAGES = 12;
constexpr int I8_SMEM_MOST = 216 * 1024;
constexpr int I8_SMS = 148;

// The sums that a CTA takes of its share of a tile's tokens, from all that share the tile's columns.
constexpr int i8_join_bytes(int bn, int split) { return split > 1 ? (bn + split - 1) / split * split * 512 : 0; }

struct I8Plan
{
	bool pair;
	int bn, split, panels, tiles_o, tiles_t;
	int smem; // for the stages
};

// A stage's bytes, how many stages there are, what a CTA asks for (from a boundary of 1024 bytes on).
constexpr int i8_stage(const I8Plan& p) { return (I8_W_BYTES + (p.pair ? p.bn / 2 : p.bn) * I8_KB) * p.panels; }
constexpr int i8_stages(const I8Plan& p)
{
	const int fit = (p.smem - 1024 - i8_join_bytes(p.bn, p.split)) / i8_stage(p);
	return fit < I8_MAX_STAGES ? fit : I8_MAX_STAGES;
}
constexpr int i8_smem(const I8Plan& p) { return i8_stages(p) * i8_stage(p) + i8_join_bytes(p.bn, p.split) + 1024; }

// Which kernel, how many tokens a tile, over how many CTAs (pairs) a tile's columns are split, one or two panels a
// stage, one CTA per SM or two (of half the memory): the least of an estimate in SM cycles. Its constants were
// fitted to 7000 timings of 180 shapes (1 to 4096 tokens, 128 to 262144 channels, 300 to 16384 columns, weights from
// HBM); the choices it makes there are 2.2 % slower than the best of all in the mean, 27 % at worst (200 x
// 4096 to 128: 4.7 us, 3.7 with half the tiles). What they stand for:
//  - a panel costs the issue of its copies and products (435 alone, 89 where two go together), its products (a pair's
//    107 + 1.75 a token, a single CTA's four of 49.3 or 44 + 0.36 a token), its bytes into an SM (64 a cycle) or, over
//    all SMs, out of L2 (10500 a cycle), or a copy's way (2670) by the panels in flight, whichever is the most;
//  - clusters of 4 and more do not fill every SM;
//  - a launch has a start and an end, and so has each CTA that runs alone on its SM after another; there is an epilogue
//    by token, and a split tile has the joining of its parts.
// Both sides, microseconds: 1 token, 6144 channels, 4096 columns: whole columns, two panels 7.5, one panel 8.8, split
// over four 8.3; 1 x 2560 x 10240: split over eight 8.1, whole 12.0; 777 x 2560 x 2048: single CTAs 7.9, pairs 8.7;
// 1024 x 6144 x 4096: pairs 22.9, single CTAs 30.4.
inline I8Plan i8_plan(int n_tok, int rows, int cols)
{
	const int n_kb = (cols + I8_KB - 1) / I8_KB;
	// how many clusters run at once with one CTA per SM and with two, by CTAs of a cluster
	static const int alone[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15}, both[9] = {0, 296, 148, 93, 71, 56, 45, 37, 33};
	const auto larger = [](double a, double b) { return a > b ? a : b; };
	I8Plan best{};
	double least = HUGE_VAL;
	// (some hundred estimates a call: what does not go by the innermost choice is worked out outside of it)
	const auto consider = [&](bool pair, int bn, int tiles_o) {
		const int tiles_t = (n_tok + bn - 1) / bn, one = I8_W_BYTES + (pair ? bn / 2 : bn) * I8_KB; // bytes of a panel
		const double tiles = (double)tiles_o * tiles_t, ends = pair ? 9600 : 3790, epilogue = (pair ? 9.4 : 18.7) * bn;
		for (int split = 1; split <= (pair ? 4 : 8) && split <= n_kb; split += split < 4 ? 1 : 2)
		{
			const int ctas = (pair ? 2 : 1) * split;
			if (split > 1 && tiles > 2 * both[ctas]) break;
			const double kb = (n_kb + split - 1) / split, join = split > 1 ? 4090 + 43.6 * bn : 0;
			const int sums = i8_join_bytes(bn, split);
			for (int two = 0; two < (pair ? 1 : 2); ++two)
			{
				const int smem = two ? 107 * 1024 : I8_SMEM_MOST, slots = two ? both[ctas] : alone[ctas], fit = std::min(I8_MAX_STAGES, (smem - 1024 - sums) / one);
				if (fit < 2 || (split > 1 && tiles > 2 * slots)) continue;
				const double waves = tiles <= slots ? 1 : tiles <= 2 * slots ? 2 : (double)(((long long)tiles + slots - 1) / slots);
				const double per_sm = two && tiles > alone[ctas] ? 2 : 1;
				const double products = pair ? 107 + 1.75 * bn : 4 * larger(49.3, 44 + 0.36 * bn) * per_sm;
				const double load = one * larger(per_sm * (1 / 64.0), (tiles < slots ? tiles : slots) * ctas * (1 / 10500.0));
				const double rest = ends + (pair || two ? 0 : 3390 * (waves - 1)) + epilogue * waves * (split > 1 ? 0.5 : 1) + join;
				for (int panels = 1; panels <= 2 && split * panels <= n_kb; ++panels)
				{
					const int stages = panels == 1 ? fit : std::min(I8_MAX_STAGES, (smem - 1024 - sums) / (2 * one));
					if (stages < panels + 1) continue;
					const double panel = larger(larger(products, load), larger(panels > 1 ? 89 : 435, 2670.0 / (panels * stages)));
					const double t = waves * kb * panel + rest;
					if (t < least) least = t, best = {pair, bn, split, panels, tiles_o, tiles_t, smem};
				}
			}
		}
	};
	const int most = n_tok < 256 ? (n_tok + 15) / 16 * 16 : 256;
	// (from the widest: of equal estimates the one with the fewest copies of the weights, 20 x 4096 to 34146 24 us, 43)
	for (int bn = most; bn >= 16; bn -= 16) consider(false, bn, (rows + 127) / 128);
	if (n_tok > 32 && rows > 128)
		for (int bn = (most + 31) / 32 * 32; bn >= 64; bn -= 32) consider(true, bn, (rows + 255) / 256);
	return best;
}

} // namespace nncu
