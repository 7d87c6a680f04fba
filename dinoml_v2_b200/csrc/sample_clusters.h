// How many CTAs have a row of the sampling together.  Host code without CUDA, so that every device's answer can be tried.
#pragma once
#include <cstdint>

namespace b200gguf {

struct SampleClusters {
  int ctas;              // of a row; 0: no size that holds one runs on the device, or that could not be found out
  int64_t at_once;       // rows whose CTAs run at once
};

// fits(c): clusters of c CTAs that run at once on the device: 0 where not one does (a part of a GPU may have fewer SMs together), negative where that could not be found out.

// 16-bit logits.  Several CTAs a row where all rows' run at once: their meetings cost what they save of a short row, or with two CTAs of a middling one.  Measured (1, 2, 4, 8 CTAs; one row, us):
// 128256 bfloat16 25.1, 20.0, 15.4, 13.6, 32000 13.2, 14.6, 13.1, 12.9, 12000 10.6, 12.6, 11.8, 12.1; 128256 values of 36 rows 28.5, 22.3, 29.7 (36 clusters of four do not run at once), 42;
// 100 rows 27.9, 41, 60, 94.
template <typename Fits> inline SampleClusters sample_clusters_16(int vocabulary, int64_t rows, int part, Fits fits) {
  for (int ctas = 8; ctas > 1; ctas /= 2) {
    if (vocabulary <= (ctas == 2 ? 53248 : 28672) || vocabulary > int64_t(ctas) * part) continue;
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
