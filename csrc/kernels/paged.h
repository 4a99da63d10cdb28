// How the work of paged attention is counted: paged_tables.cu makes the prefix sums of a step,
// paged_attention.cu cuts them into equal ranges. ops/paged.py holds the same two numbers for the oracle.
#pragma once

namespace hrm {

constexpr int kUnitKeys = 128;  // keys of one unit: 32 for each of a CTA's 4 warps
// What starting and finishing a (request, head) costs, in units: first loads, merging the warps, writing.
constexpr int kPairCost = 3;

}  // namespace hrm
