"""Sizes of 8-bit products (rows, columns, channels) and scores (maps, height, width, channels) that reach each kernel on 256 compute units."""
FEW = [(300, 40, 128), (70, 130, 112), (70, 300, 144), (500, 90, 1024), (9000, 20, 400)]    # the last three deal the blocks to four waves from 3 blocks on
SHORT = [(9000, 300, 128), (9001, 301, 112), (16500, 65, 64)]
LONG = [(9000, 300, 144), (9001, 301, 256), (9000, 300, 272), (8200, 130, 1024)]
PRODUCTS = FEW + SHORT + LONG
SCORES_FEW = [(2, 12, 23, 128), (3, 9, 7, 256)]
SCORES_LDS = [(64, 12, 23, 128), (300, 17, 31, 128), (260, 24, 30, 128), (64, 12, 23, 256), (260, 17, 31, 256)]
SCORES = SCORES_FEW + SCORES_LDS
