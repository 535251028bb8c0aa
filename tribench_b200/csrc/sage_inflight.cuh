// sage_inflight.cuh — which asynchronous copies a warp has issued and may have to wait for.
//
// A block's shared memory is another block's as soon as it has left. Where every wait of the block was
// served, every copy has landed: those who use it waited for it. Where one ran out, a warp that issued
// bulk copies still has to wait for the last one into each slot (earlier ones had landed before their
// slot was reused), by the parity of the barrier phase that it completes. Plain C++, so that the
// bookkeeping runs on the host too.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define SAGE_BOTH __host__ __device__ __forceinline__
#else
#define SAGE_BOTH inline
#endif

namespace sage {

struct CopyLedger {
  uint32_t issued = 0;  // bit s: the last copy into slot s went to this ledger's barriers
  uint32_t parity = 0;  // bit s: the parity of its phase
  SAGE_BOTH void note(int s, uint32_t phase) {
    issued |= 1u << s;
    parity = (parity & ~(1u << s)) | ((phase & 1u) << s);
  }
  // Another warp completes the next phase of slot s's barrier: this ledger's has long completed, and its
  // parity would name a phase to come.
  SAGE_BOTH void forget(int s) { issued &= ~(1u << s); }
  SAGE_BOTH bool pending(int s) const { return (issued >> s) & 1u; }
  SAGE_BOTH uint32_t phase(int s) const { return (parity >> s) & 1u; }
};

// The copies of values that the chunk kernel's producer issues: on `raw` barriers where another warp
// still has to work on the tile before it is full, else on the `full` ones. `raw` phases count the raw
// tiles of a slot.
struct ValueCopies {
  CopyLedger full, raw;
  uint32_t raw_next = 0;  // bit s: parity of slot s's next raw phase
  SAGE_BOTH void note(int s, uint32_t phase, bool is_raw) {
    if (is_raw) {
      raw.note(s, raw_next >> s);
      raw_next ^= 1u << s;
      full.forget(s);
    } else {
      full.note(s, phase);
    }
  }
};

// The last copies of a ring of `slots` barriers on which tile j completes phase j / slots, after `tiles` of them.
SAGE_BOTH CopyLedger ring_copies(int tiles, int slots) {
  CopyLedger c;
  for (int j = tiles > slots ? tiles - slots : 0; j < tiles; ++j) c.note(j % slots, j / slots);
  return c;
}

}  // namespace sage
