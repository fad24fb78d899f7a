/* Who quantises what in the product that quantises its own rows (gb_gemm_blocks.cu), as plain arithmetic that a host program can
 * compile as well.
 *
 * The blocks of K that a CTA multiplies are numbered through, over all of its tiles: slab 0, 1, 2, ...  Slab n lies in stage n % kStages of
 * the operand ring, and its rows may be written there once the multiplication of slab n - kStages has freed the stage.  A
 * barrier tells the phase that a wait asks for from the one before or behind it only, so whoever waits for a stage has to have
 * seen every earlier phase of it.  Slabs are not multiplied in order (two issuers take them in turn, each as its operands land): that a
 * later slab is done says nothing about an earlier one.  So a group of lanes has one slab of every kSlabsAStep by its running number,
 * over the ends of tiles too, and as the stages are a multiple of that, its slabs come round to the same stages each time, and it waits
 * for every phase of them. */
#pragma once

namespace gb_row_ring {

constexpr int kStages = 8, kSlabsAStep = 4;
static_assert(kStages % kSlabsAStep == 0, "a group of lanes meets every phase of its stages");

/* Groups of eight lanes, of which kSlabsAStep * rows work. */
constexpr bool works(int group, int rows) { return group < kSlabsAStep * rows; }
constexpr int first_slab(int group, int rows) { return group / rows; }
constexpr int row(int group, int rows) { return group % rows; }

}  // namespace gb_row_ring
