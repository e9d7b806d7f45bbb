// Host build of the check of an item's note (csrc/cache4_layout.h) for tests/test_cache4_edges_host.py.
#include "cache4_layout.h"

extern "C" int ra_host_cache_note_holds(int first, int last, int ctas) { return ra::cache_note_holds(first, last, ctas); }
