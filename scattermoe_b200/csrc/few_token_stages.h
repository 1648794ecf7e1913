// How the streaming kernels of few_token.cu cut their ring of shared memory into stages: host arithmetic on its own, so that it can be
// checked without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define SMOE_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define SMOE_HOST_DEVICE inline
#endif

namespace smoe {
namespace ft {

constexpr int MAX_STAGES = 16;
constexpr int STAGE_GROUPS = 4;                // groups of 8 slots of a job, at most
constexpr int GROUP_BYTES = 1024;              // the rows of 8 slots, 64 of K (128 bytes) each
constexpr int RING_SLACK = 2048;               // ldmatrix reads whole 16-row blocks: past a box of fewer rows (never used, but inside the ring)
constexpr int MAX_STAGE_BYTES = 48 * 1024;
constexpr int MAX_WEIGHT_BYTES = 32 * 1024;    // of a stage of the up-projection

struct Stages {
  int stages, stage_bytes;
  int steps_of[4][STAGE_GROUPS];               // steps of K of a stage: 1, 2, 3-4, 5-8 boxes wide x a job of 1-8, 9-16, 17-24, 25-32 slots
};

// Class of a round that is `boxes` boxes wide.
SMOE_HOST_DEVICE int width_class(int boxes) { return boxes <= 2 ? boxes - 1 : (boxes <= 4 ? 2 : 3); }

// Stages of up to 48 KB, weights and beside them the rows of the job's slots: four, or as many more (a multiple of the turns) as
// `ring` bytes hold where the whole of K needs less. How much less goes by the slots an expert has when a token's experts differ (T at
// most); but a token may name an expert more than once, so the largest job has up to T k slots, and a stage holds one step of that as
// well. False where the stages cannot be made.
inline bool make_stages(Stages* out, bool up, int ring, int box_bytes, int blocks, int T, int k, int turns) {
  auto groups_of = [](int slots) { return slots < 8 * STAGE_GROUPS ? (slots + 7) / 8 : STAGE_GROUPS; };
  const int usual_groups = groups_of(T), most_groups = groups_of(T * k);
  out->stage_bytes = (ring - RING_SLACK) / 4 / 1024 * 1024;
  if (out->stage_bytes > MAX_STAGE_BYTES) out->stage_bytes = MAX_STAGE_BYTES;
  const int least = box_bytes + most_groups * GROUP_BYTES;
  int64_t whole = static_cast<int64_t>(blocks) * (box_bytes + usual_groups * GROUP_BYTES);
  if (whole < least) whole = least;
  if (!up && whole < out->stage_bytes) out->stage_bytes = static_cast<int>(whole);
  if (out->stage_bytes < least) return false;
  out->stages = (ring - RING_SLACK) / out->stage_bytes;
  out->stages = (out->stages > MAX_STAGES ? MAX_STAGES : out->stages) / turns * turns;
  if (out->stages < turns) return false;
  for (int c = 0; c < 4; ++c)
    for (int g = 0; g < STAGE_GROUPS; ++g) {
      const int boxes = 1 << c;      // the most of their class; never more than 32 KB of weights in the up-projection's rounds
      const bool reached = g < most_groups && boxes * box_bytes <= (up ? MAX_WEIGHT_BYTES : box_bytes);
      int steps = out->stage_bytes / (boxes * box_bytes + (g + 1) * GROUP_BYTES);
      if (up && steps > MAX_WEIGHT_BYTES / (boxes * box_bytes)) steps = MAX_WEIGHT_BYTES / (boxes * box_bytes);
      if (steps < 1 && reached) return false;
      const int stages_of_k = steps < 1 ? blocks : (blocks + steps - 1) / steps;
      out->steps_of[c][g] = (blocks + stages_of_k - 1) / stages_of_k;
    }
  return true;
}

}  // namespace ft
}  // namespace smoe
