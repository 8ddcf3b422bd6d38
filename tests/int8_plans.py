"""Shapes (M, K, N) of products of 8-bit rows by the kernel and the cut of k that they take (names of dmf_int8_linear_kernel_name): odd
sizes, so that tiles are ragged, and for the CTA pairs results that leave by TMA (N a multiple of 8) and results that cannot."""

PLANS = {
    "int8_gemm_few_kernel<16>": [(1, 16, 131), (209, 130, 54)],
    "int8_gemm_few_kernel<16>, k over 2 CTAs": [(1, 1750, 3755), (6, 2577, 6885), (7, 4305, 5012)],
    "int8_gemm_few_kernel<16>, k over 4 CTAs": [(1, 911, 539), (113, 1290, 186)],
    "int8_gemm_few_kernel<16>, k over 8 CTAs": [(1, 987, 133), (2, 1587, 501), (35, 4700, 261)],
    "int8_gemm_few_kernel<32>": [(17, 16, 10329), (1218, 18, 134), (53, 21, 5073)],
    "int8_gemm_few_kernel<32>, k over 2 CTAs": [(20, 2460, 4770), (660, 2798, 134), (401, 2601, 336)],
    "int8_gemm_few_kernel<32>, k over 4 CTAs": [(18, 2440, 2459), (309, 2711, 146), (305, 4659, 247), (148, 2468, 424)],
    "int8_gemm_few_kernel<32>, k over 8 CTAs": [(151, 5162, 131), (18, 5212, 1277), (64, 4673, 586)],
    "int8_gemm_few_kernel<64>": [(2386, 298, 132), (410, 807, 1675)],
    "int8_gemm_few_kernel<64>, k over 2 CTAs": [(1199, 4266, 131), (35, 5059, 4742)],
    "int8_gemm_few_kernel<64>, k over 4 CTAs": [(599, 6277, 139), (36, 7027, 2329), (445, 6586, 280)],
    "int8_gemm_few_kernel<64>, k over 8 CTAs": [(625, 11789, 1), (704, 12882, 35), (639, 12113, 8)],
    "int8_gemm_pair_kernel<128>": [(9707, 17, 1), (10054, 18, 8), (2049, 144, 776), (19000, 64, 257)],
    "int8_gemm_pair_kernel<192>": [(280, 17, 7062), (14151, 17, 141), (14103, 22, 144), (8200, 256, 1152)],
    "int8_gemm_pair_kernel<256>": [(274, 131, 8345), (288, 139, 8584), (2748, 153, 1432), (4541, 1318, 6302), (4100, 1153, 4608)],
    "int8_gemm_pair_kernel<256>, narrow end": [(19942, 885, 1), (19674, 1048, 8), (20000, 130, 1100), (4000, 1152, 1152)],
}
