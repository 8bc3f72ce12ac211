// Host check of how the places of a linear attention call share the batch's
// tokens: argv: tokens, batch. Prints the tokens counted over all places, the
// most that one has, and the first place that has one out of order (-1: none).
#include <cstdio>
#include <cstdlib>

#include "layer.h"

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  const long long tokens = atoll(argv[1]), batch = atoll(argv[2]);
  long long total = 0, most = 0, bad = -1;
  for (long long place = 0; place < jv::linear_chunks(tokens, batch); ++place) {
    const long long n = jv::rows_at((int)place, (int)tokens);
    if (n < 0 || (n && place * jv::kChunk != total)) bad = bad < 0 ? place : bad;
    total += n, most = n > most ? n : most;
  }
  printf("%lld %lld %lld\n", total, most, bad);
  return 0;
}
