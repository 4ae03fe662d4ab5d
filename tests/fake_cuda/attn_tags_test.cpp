/* The rule of attn_tags.h: in no launch does a word that another launch wrote carry this one's
 * number, whichever words the launches between have written.  With counters of few rounds every
 * start and every gap is gone through, and a few turns of random launches; at the full width the
 * clearing rounds are looked up.  With a counter that wraps through 0, and without the clearing, the
 * same launches do find such words. */
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "attn_tags.h"

static uint64_t state = 1;
static unsigned draw(unsigned n) {
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    return (unsigned)((state >> 33) % n);
}

/* a word that is written in the first launch, and in none of the `gap` after it */
static bool passes(unsigned start, unsigned gap, unsigned last) {
    unsigned counter = start, word = 0;
    for (unsigned i = 0; i <= gap; i++) {
        counter = apus::ad_round_after(counter, last);
        if (counter == 0 || counter > last) return true;      /* what no word may be told from */
        if (i && word == counter) return true;
        if (apus::ad_round_clears(counter, last)) word = 0;
        if (!i) word = counter;
    }
    return false;
}

static long stale(bool mended, unsigned last, long launches) {
    const int WORDS = 16;
    unsigned words[WORDS] = {}, counter = 0;
    long wrong = 0;
    for (long n = 0; n < launches; n++) {
        counter = mended ? apus::ad_round_after(counter, last) : counter == last ? 0 : counter + 1;
        const bool clears = mended && apus::ad_round_clears(counter, last);
        for (int w = 0; w < WORDS; w++) {
            /* what a CTA may see that asks before the words are cleared or written */
            wrong += words[w] == counter;
            if (clears) words[w] = 0;
            if (draw(1u << w) == 0) words[w] = counter;       /* w: written every 2^w launches */
        }
    }
    return wrong;
}

int main() {
    long wrong = 0, found = 0;
    for (unsigned last : {7u, 15u, 255u, 1000u, 1023u})
        for (unsigned start = 0; start <= last; start++)
            for (unsigned gap : {last - 1, last, last + 1, 2 * last, 2 * last + 1})
                wrong += passes(start, gap, last);
    for (unsigned last : {255u, 1023u, 65535u}) {
        wrong += stale(true, last, 40 * (long)last + 7);
        found += stale(false, last, 40 * (long)last + 7) != 0;
    }
    unsigned clears[2], n = 0;
    for (unsigned r : {0x3fffffffu, 0x40000000u, 0x40000001u, 0xbffffffeu, 0xbfffffffu, 0xc0000000u,
                       0xffffffffu, 0u, 1u, 2u})
        if (apus::ad_round_clears(r)) {
            if (n < 2) clears[n] = r;
            n++;
        }
    const bool full = n == 2 && clears[0] == 0x40000000u && clears[1] == 0xbfffffffu &&
                      apus::ad_round_after(0) == 1 &&
                      apus::ad_round_after(0xfffffffeu) == 0xffffffffu &&
                      apus::ad_round_after(0xffffffffu) == 1;
    printf("%ld stale words, %ld of 3 counters without the rule have some, full width %d\n", wrong,
           found, full);
    return wrong != 0 || found != 3 || !full;
}
