// Bit map of a row's listed classes: the class `base + d` has bit BIT0 + d.  base is a vector's first class, so a vector's
// bits lie within one byte; the BIT0 bits in front are for the classes before the row's first whole vector.  Host code too.
#pragma once

constexpr int BIT0 = 16;
// Words that hold the bits of `classes` classes from base on.
constexpr int map_words(int classes) { return (BIT0 + classes + 31) / 32; }

// Wide rows have a map of SEG classes at a time: the words of its first segment, which no later one exceeds.
constexpr int SEG = 131072, SEG_WORDS = map_words(SEG);
constexpr int segment_words(int ncls) { return map_words(ncls < SEG ? ncls : SEG); }
static_assert(segment_words(1 << 20) <= SEG_WORDS && segment_words(SEG) <= SEG_WORDS && segment_words(1) <= SEG_WORDS, "the map holds every segment");
