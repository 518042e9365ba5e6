/* embed.S -- places the gfx950 code objects (FFT, and the sequence filters for
 * each element type) inside libferrum_gpu.so so the HIP backend can hand them
 * to hipModuleLoadData without touching the file system (FG_HSACO_PATH and
 * FG_SSM_*_PATH are set by the Makefile). */
    .section .rodata.fg_fft_code_object,"a",@progbits
    .p2align 12
    .globl fg_fft_code_object_start
    .hidden fg_fft_code_object_start
fg_fft_code_object_start:
    .incbin FG_HSACO_PATH
    .globl fg_fft_code_object_end
    .hidden fg_fft_code_object_end
fg_fft_code_object_end:
    .byte 0

#define FG_EMBED(name, path)                        \
    .section .rodata.fg_##name##_code_object,"a",@progbits; \
    .p2align 12;                                    \
    .globl fg_##name##_code_object_start;           \
    .hidden fg_##name##_code_object_start;          \
fg_##name##_code_object_start:                      \
    .incbin path;                                   \
    .globl fg_##name##_code_object_end;             \
    .hidden fg_##name##_code_object_end;            \
fg_##name##_code_object_end:                        \
    .byte 0
FG_EMBED(ssm_f32, FG_SSM_F32_PATH)
FG_EMBED(ssm_bf16, FG_SSM_BF16_PATH)
FG_EMBED(ssm_f16, FG_SSM_F16_PATH)
    .section .note.GNU-stack,"",@progbits
