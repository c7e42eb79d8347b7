// The order in which the roles of extend_kernel take the steps of a segment. Plain functions of the
// segment's counts, without CUDA, so that the barrier protocol can be run on the host too.
//
// An mbarrier wait names a phase by its parity only: it passes when the phase before the named one
// is the last that completed, one phase early, and blocks for good when the one behind it has
// completed as well. So a role may wait for phase p of a barrier only if it knows that phase p - 1
// has completed, and if phase p + 1 cannot complete without it.
//   s_full[b]     Step n is waited for by its own chain. Q K^T of step n - kSBufs has completed: the
//                 chain's last step is at most kSBufs steps back inside a segment. From one segment
//                 to the next chain 1, which has the last step of a two-tile segment, and both chains
//                 of a joined one know that all of it has completed. Chain 0 of another two-tile
//                 segment knows by o_full[0] that every Q K^T issued before its last P V has: all of
//                 the segment but at most kSBufs - 1 steps, since the second tile sees at most one
//                 key tile more than the first. Where the first tile sees none (more rows than keys,
//                 or a share that starts behind its keys), chain 0 would wait for nothing, and two
//                 such segments in a row would put it two phases behind: they are joined.
//   p_half[b]     128 arrivals of the chain that owns the step, which waited for s_full[b] first; the
//                 MMA lane waits for each of them.
//   o_full[c]     Once per segment in which chain c has steps, and waited for each time.
//   x_ready/done  Once per joined segment, waited for each time by the other chain.
//   q, k, v       Rings whose two sides wait for every phase. A chain also waits for the v_empty of its
//                 previous step's tile, see PrevPv.
//   scale_full[s] The converter of K writes a tile's scales before the tile, so s_full of the step says that
//                 they are there; their place is taken again only once the readers are done (kScaleSlots).
//   code_full[s]  The tiles of one place belong to K and V by turns, and copies land in any order: a
//                 converter that waits for its tile knows nothing of the one before, which is the
//                 other's. So it waits for that tile's release first. Its own comes next, so the
//                 release cannot be a phase further.
#pragma once

#ifdef __CUDACC__
#define FLB_HD __host__ __device__ __forceinline__
#else
#define FLB_HD inline
#endif

namespace flb {

// A segment's steps: chain c works on count(c) key tiles.
struct Steps {
  bool dual;            // the tokens fit in one tile, whose key tiles the chains share
  int count0, count1;

  FLB_HD int count(int c) const { return c == 0 ? count0 : count1; }

  // The place of chain c's j-th key tile among the segment's.
  FLB_HD int place(int c, int j) const { return dual ? 2 * j + c : j; }
  // The chains take turns while both have steps (chain 0 runs out first in a two-tile item): the
  // place of chain c's j-th step among the steps of both.
  FLB_HD int order(int c, int j) const { return dual || j < count0 ? 2 * j + c : count0 + j; }

  // Steps in which the chains take turns, and the chain of step i.
  FLB_HD int paired() const { return dual ? count0 + count1 : 2 * count0; }
  FLB_HD int chain(int i) const { return i < paired() ? i & 1 : 1; }
  // The last step of the chain that does not have the segment's last one (none: negative).
  FLB_HD int other_last() const { return paired() - 2; }

  // The chains meet at the segment's end.
  FLB_HD bool joined() const { return dual || count0 == 0; }
};

// Place of the i-th K or V tile of codes among the 2 n of a segment, in the producer's order: K 0,
// K 1, V 0, K 2, V 1, ..., V n - 1.
FLB_HD int code_place(bool is_v, int i, int n) {
  return is_v ? (i + 1 < n ? 2 * i + 2 : 2 * i + 1) : (i > 0 ? 2 * i - 1 : 0);
}

}  // namespace flb
