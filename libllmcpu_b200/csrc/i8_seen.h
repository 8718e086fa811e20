// i8_seen.h -- what the checks of the 8-bit products remember (k_i8.cu): of
// each stream how many waits that ran out its last check saw. Plain C++.
#pragma once

#include <mutex>
#include <vector>

namespace nncu
{

// The device counts the waits that ran out and nobody takes them off the
// count, so that one stream's check hides none from another's. Nothing is
// kept until the first one.
class I8Seen
{
public:
	// Whether `count` says of more than the last check of this stream (by its number, which no other one ever has) saw.
	bool more(int device, unsigned long long stream, unsigned count)
	{
		if (count == 0) return false;
		std::lock_guard<std::mutex> lk(mu_);
		for (Entry& e : seen_)
			if (e.device == device && e.stream == stream)
			{
				const bool more = e.count != count;
				e.count = count;
				return more;
			}
		seen_.push_back({device, stream, count});
		return true;
	}

private:
	struct Entry
	{
		int device;
		unsigned long long stream;
		unsigned count;
	};
	std::mutex mu_;
	std::vector<Entry> seen_;
};

} // namespace nncu
