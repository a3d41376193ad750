"""Layers whose products run through all of the streaming loop of the expert layer's larger form: chunks of columns, more rounds of row tiles
than the shared memory has room for, several row tiles a round.  What each is for is held by tests/test_w4_plan_cpu.py against the
library's own planning; tests/test_moe_w4_runs_gpu.py runs them."""

# T, D, I, E, k, type, group, zero (types: 0 bf16, 1 f16), and what its up and its down products must show on 148 SMs
RUNS = [
    # up: two chunks, more rounds than room and a last set of one or two; down: two chunks of four rounds, the last unit without its second tile
    ((29, 2176, 3856, 1, 1, 0, 32, True), {"chunks": 2, "past_room": True}, {"chunks": 2, "rounds": 3}),
    # down: the same over the two-term activations; up: two chunks of seven rounds, two units a warp
    ((29, 7720, 2056, 1, 1, 1, 64, True), {"chunks": 2, "rounds": 6}, {"chunks": 2, "past_room": True}),
    # down: two chunks with three row tiles a round, warps left over, a last row tile of 8 rows
    ((25, 3576, 1032, 4, 4, 0, 128, False), {"rounds": 2}, {"chunks": 2, "slots": 2, "rounds": 3}),
    # two chunks for runs of a single row tile
    ((20, 4232, 136, 2, 2, 0, 128, True), {"chunks": 2}, {"slots": 2}),
    ((20, 136, 2312, 2, 2, 1, 128, False), {"slots": 2}, {"chunks": 2}),
]
SMS = 148
