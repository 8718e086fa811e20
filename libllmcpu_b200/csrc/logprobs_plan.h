// logprobs_plan.h -- which kernel reads rows of logits, and how many CTAs share
// a row (k_logprobs.cu). Plain C++.
#pragma once

#include <cmath>

namespace nncu
{

constexpr int LP_CLUSTER = 8; // the most CTAs that share a row
constexpr int LP_WIDE = 512, LP_NARROW = 256; // threads of a CTA: where rows are few, and where they are many
// CTAs per SM.
constexpr int lp_ctas(int threads, bool ahead) { return threads == LP_WIDE ? 2 : ahead ? 4 : 5; }

struct LpPlan
{
	bool wide, ahead;
	int parts; // CTAs that share a row
};

// The least of an estimate, in SM cycles: the waves that the CTAs make of what the GPU holds at once (clusters do not
// fill every SM) times a CTA's start and end and its share, at a pace of its own or, with others on its SM, at a share
// of the SM's. Its constants were fitted to 2600 timings (1 to 2000 rows of 5000 to 162275 logits, from HBM); its
// choices are 0.3 % slower there than the best of all in the mean, 8 % at worst. Both sides, microseconds, with 5
// alternatives: 64 rows of 151936: wide CTAs, four a row 13.6, narrow ones 17.1; 1 x 262144: eight wide CTAs 6.9, one
// 20.4; 450 rows of 43807: narrow CTAs 24.3, with loads ahead 20.2, wide ones 25; 700 rows: 29.2 and 32.8.
inline LpPlan lp_plan(long long n, int n_vocab, bool top)
{
	struct Kind
	{
		bool wide, ahead;
		double ends, top_ends, join, top_join, pace; // cycles a CTA, and a logit
		int all_of_8; // SMs that clusters of eight fill
	};
	const Kind kinds[] = {{true, true, 3310, 2170, 443, 190, 0.098, top ? 124 : 132},
	                      {false, true, 3560, 2210, 183, 290, 0.192, top ? 132 : 136},
	                      {false, false, 3520, 4150, 320, 90, 0.259, 132}};
	LpPlan best{};
	double least = HUGE_VAL;
	for (const Kind& k : kinds)
		for (int i = 0, parts = 1; parts <= LP_CLUSTER; ++i, parts *= 2)
		{
			const int filled[] = {148, 148, 142, k.all_of_8}; // SMs that clusters of 1, 2, 4, 8 fill
			const double slots = filled[i] * lp_ctas(k.wide ? LP_WIDE : LP_NARROW, k.ahead), ctas = (double)n * parts;
			const double beside = std::fmax(1.0, std::fmin(ctas, slots) / 148);
			double ends = k.ends;
			if (top) ends += k.top_ends;
			if (parts > 1) ends += k.join + (top ? k.top_join : 0);
			const double pace = std::fmax(k.pace, 0.045 * beside);
			const double t = std::ceil(ctas / slots) * (ends * std::fmax(1.0, 0.145 * beside) + pace * n_vocab / parts);
			if (t < least) least = t, best = {k.wide, k.ahead, parts};
		}
	return best;
}

} // namespace nncu
