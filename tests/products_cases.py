"""Sizes at which every product kernel and form of the operator programs runs
its main loop into its steady state: more steps than registers or rings hold,
k split over several workgroups, partial tiles beside whole ones. The GPU
tests compare them with 64 bits; a CPU test shows that they cover every kernel."""

# M, K, N of few rows: steps of 32 k over 8 waves and P workgroups; the last
# step short, the last chunk uneven, strips partial, P = 1 with long k (257 strips).
FEW = [(1, 257, 40), (1, 4099, 640), (16, 1031, 333), (16, 4099, 8001), (17, 1032, 640), (17, 4099, 8001), (33, 4096, 200),
       (33, 4100, 8008), (64, 4099, 131), (64, 4099, 8001), (5, 2600, 16448), (30, 2600, 16451), (64, 1100, 16391)]

# Planes (rows, columns) of odd rows above 2^20 results, below and above 128
# tiles of 128 x 128, and one below (split); REDUCTION_ODD is their k.
ODD_PLANES = [(1001, 1501), (1537, 1801), (500, 769)]
REDUCTION_ODD = 1003

# Planes of whole chunks, one for each form of a plain product and of a pair
# (whose tiles have half the columns), and two whose k is split.
WHOLE_PLANES = [(200, 264), (72, 14560), (2056, 520), (2056, 1032), (2056, 2056), (3080, 1032), (3080, 2056), (3592, 1288),
                (3592, 2568)]
REDUCTION_WHOLE = 1096  # 17 turns of 64 and 8 left over
