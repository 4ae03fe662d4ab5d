/*
 * attn_tags.h — the numbers of decode attention's rounds (attn_decode.cuh), which are the tags of
 * the words that its CTAs exchange, and when those words are cleared.  Plain C++, so that a test
 * without a GPU can take a counter through its whole range.
 *
 * Every launch is a round, and the next one's number follows on the one before it: 1 to `last`, and 1
 * again (0 is what words hold that nobody has written, or that were cleared).  A word that was written
 * `last` launches ago and not since, in a part that few launches have, would pass as this one's: half
 * a day of launches of 12 us.  So twice in a turn a launch clears all words before it writes its
 * own.  Between a round and the next one of its number there is always such a launch: they are
 * half a turn apart, and one that writes the word itself has cleared it before.
 */
#pragma once
#include "exact_codes.h"

namespace apus {

/* the number after this one; a new counter is 0.  (last: 2^32 - 1, but in tests) */
APUS_HD unsigned ad_round_after(unsigned round, unsigned last = 0xffffffffu) {
    return round < last ? round + 1 : 1;
}
/* (a quarter and three quarters through: not the first launches of a process) */
APUS_HD bool ad_round_clears(unsigned round, unsigned last = 0xffffffffu) {
    return round == last / 4 + 1 || round == last / 4 + last / 2 + 1;
}

}  // namespace apus
