// How many CTAs have a row of the sampling together.  Host code without CUDA, so that every device's answer can be tried.
#pragma once
#include <cstdint>

namespace b200gguf {

struct SampleClusters {
  int ctas;              // of a row; 0: no size that holds one runs on the device, or that could not be found out
  int64_t at_once;       // rows whose CTAs run at once
};

// fits(c): clusters of c CTAs that run at once on the device: 0 where not one does (a part of a GPU may have fewer SMs together), negative where that could not be found out.

// 16-bit logits.  Several CTAs a row where all rows' run at once: their meetings cost what they save of a short row.  Measured (bfloat16, top_p, us a launch; 1, 2, 4, 8 CTAs a row):
//   one row of 20000 11.2, 12.8, 11.8, 12.0; 24000 12.6, 14.4, 13.0, 12.8; 28672 13.1, 14.7, 13.3, 13.0; 40000 12.9, 13.9, 12.0, 12.2; 128256 23.5, 19.2, 15.3, 13.6
//   33 rows of 24000 12.9, 14.4, 13.2, -; 28672 13.8, 14.9, 13.6, -; 40000 14.6, 15.6, 13.7, -; 128256 27.5, 22.3, 16.1, 40.5 (clusters of eight run in three turns then)
//   74 rows of 45056 15.7, 16.7, -, -; 48000 16.5, 16.5; 50257 18.1, 17.6; 56000 18.1, 17.4; 128256 28.4, 23.0, 46.5, 67.9
// So four and eight from 28672 on, two where one CTA would count in a second turn (8 * 6144 values).
// A part holds no more values than a 16-bit count: two parts end at 131056, four at 262112, and behind that fewer rows run with several CTAs (40 rows of 128256 22.2, of 131072 27.5, of 151936
// 30.8; 20 rows of 262112 21.8, of 262144 46.9).
template <typename Fits> inline SampleClusters sample_clusters_16(int vocabulary, int64_t rows, int part, Fits fits) {
  for (int ctas = 8; ctas > 1; ctas /= 2) {
    if (vocabulary <= (ctas == 2 ? 49152 : 28672) || vocabulary > int64_t(ctas) * part) continue;
    const int64_t n = fits(ctas);
    if (n < 0) return {0, 0};
    if (rows <= n) return {ctas, n};
  }
  const int64_t n = fits(1);
  return n > 0 ? SampleClusters{1, n} : SampleClusters{0, 0};
}

// float32 logits.  As many CTAs a row as let all rows' run at once, of 1024 values at least, and no fewer than hold a row (`part` values each).  Measured (1, 2, 4, 8 CTAs; us): 50001 values of one
// row -, 38, 28, 23, of 18 rows -, 40, 29, 44, of 256 -, 150, 215, 370; 20000 values of one row 31, 25, 21, 20, of 74 33, 27, 58, 90; 300 of one row 12.1, 13.6, 14.1, 14.6.
template <typename Fits> inline SampleClusters sample_clusters_32(int vocabulary, int64_t rows, int part, Fits fits) {
  int least = 1;
  while (least < 8 && int64_t(least) * part < vocabulary) least *= 2;
  for (int ctas = 8; ctas >= least; ctas /= 2) {
    const int64_t n = fits(ctas);
    if (n < 0) return {0, 0};
    if (n > 0 && (ctas == least || (rows <= n && vocabulary / ctas > 1024))) return {ctas, n};
  }
  return {0, 0};
}

}  // namespace b200gguf
