/* Embeds the gfx950 code objects (built by hipcc --genco) into libbrik.so. */
    .section .rodata.brik_hsaco, "a"
    .balign 4096
    .globl brik_hsaco_begin
    .type brik_hsaco_begin, @object
brik_hsaco_begin:
    .incbin BRIK_HSACO_PATH
    .globl brik_hsaco_end
brik_hsaco_end:
    .byte 0
    .balign 4096
    .globl brik_attn_hsaco_begin
    .type brik_attn_hsaco_begin, @object
brik_attn_hsaco_begin:
    .incbin BRIK_ATTN_HSACO_PATH
    .byte 0
    .balign 4096
    .globl brik_moe_hsaco_begin
    .type brik_moe_hsaco_begin, @object
brik_moe_hsaco_begin:
    .incbin BRIK_MOE_HSACO_PATH
    .byte 0
    .section .note.GNU-stack, "", @progbits
