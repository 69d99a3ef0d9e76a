"""Sizes at which every product kernel and form of the operator programs runs
its main loop into its steady state: more steps than registers or rings hold,
k split over several workgroups, partial tiles beside whole ones. The GPU
tests compare them with 64 bits; a CPU test shows that they cover every kernel."""

# M, K, N of few rows: steps of 32 k over 8 waves and P workgroups; the last
# step short, the last chunk uneven, strips partial, P = 1 with long k (257 strips).
FEW = [(1, 257, 40), (1, 4099, 640), (16, 1031, 333), (16, 4099, 8001), (17, 1032, 640), (17, 4099, 8001), (33, 4096, 200),
       (33, 4100, 8008), (64, 4099, 131), (64, 4099, 8001), (5, 2600, 16448), (30, 2600, 16451), (64, 1100, 16391)]
