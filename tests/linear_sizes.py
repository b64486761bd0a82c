"""Sizes (rows, inner, outer) at which the linear layer is tested."""

SIZES = [(1, 1, 1), (5, 3, 2), (1, 64, 256), (8, 256, 1000), (64, 32, 32), (257, 45, 100), (130, 64, 256), (300, 5, 32),
         (300, 32, 3), (77, 130, 40), (65, 256, 64), (33, 250, 1100), (2500, 16, 24), (1, 1100, 7), (40, 1000, 200),
         (3, 2000, 31), (513, 129, 33), (700, 600, 130)]

# each number of blocks of the contraction for which the weights stay in LDS, in
# 16-bit types and in float32, a slice of the columns and several
RESIDENT = [(1025, 20, 5), (1300, 50, 70), (1100, 90, 129), (2050, 120, 64), (1500, 150, 300), (1030, 180, 33),
            (1090, 210, 100), (1500, 256, 610), (1024 + 7, 16, 1), (1111, 96, 40), (1200, 112, 8)]
# weights streamed: each number of column blocks of a slice
STREAMED = [(1025, 257, 20), (1100, 300, 50), (1600, 1000, 96), (1040, 333, 120), (1300, 270, 160), (1026, 520, 190),
            (1025, 1000, 200), (1090, 264, 256), (1200, 290, 290), (2200, 600, 3)]

# weight gradients that one workgroup holds (each of its shapes), rows from less than
# a block to several a workgroup
ONE_PASS = [(7, 64, 256), (33, 60, 250), (2100, 33, 200), (9000, 64, 96), (500, 128, 256), (4500, 70, 130), (40, 256, 64),
            (3000, 250, 50), (700, 256, 128), (5000, 129, 65), (20000, 8, 3)]
