// CPU check of a reader's turns in a ring whose producer stops: every tile that begins or ends behind the last block that came has to
// know it, whatever the barriers' bits say by then.  Built and run by tests/test_ring_turn.py.
#include <cstdio>

#include "../mixture-of-kittens_b200/csrc/ring_turn.cuh"

constexpr int kStages = 4;

// Barriers of one bit: stage s has completed as many phases as blocks of it came, and a wait for a parity passes when the phase in
// progress has the other one.
struct Barriers {
    int done[kStages] = {0, 0, 0, 0};
    bool passed(uint32_t stage, uint32_t parity) const { return (done[stage] & 1u) != parity; }
};

int main() {
    for (int tile_blocks = 1; tile_blocks <= 9; ++tile_blocks)
        for (int served = 0; served <= 40; ++served) {
            Barriers bars;
            mok::RingTurn<kStages> turn;
            int block = 0;
            for (int tile = 0; tile < 20; ++tile) {
                const int end = block + tile_blocks;
                for (int left = tile_blocks; left > 0; --left, ++block) {
                    if (block < served) ++bars.done[block % kStages];   // comes in time
                    if (!turn.next([&](uint32_t stage, uint32_t parity) { return bars.passed(stage, parity); })) break;
                }
                if (turn.ok != (end <= served)) {
                    std::printf("FAILED: tiles of %d blocks, %d blocks came, tile %d is taken for %s\n", tile_blocks, served, tile,
                                turn.ok ? "whole" : "broken");
                    return 1;
                }
                if (!turn.ok) block = end;
            }
        }
    std::printf("ok\n");
    return 0;
}
