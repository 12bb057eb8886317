/*
 * cc1d_checkpoint.h — C ABI of the 8-bit activation checkpoint of libcc1d.so (B200, sm_100a).
 *
 * The convolution's backward needs x again.  These calls keep it in 8 bits instead: each value as
 * e4m3 (4 exponent bits, 3 mantissa bits), with one power-of-two scale for each 32 neighbours
 * along the contiguous axis of x: the least power of two that brings all of them within e4m3's
 * largest number, 448.  Rounding is to the nearest, ties to even: a kept value is off by at most
 * 2^-4 of itself (2^-10 times its scale for values below 2^-6 times the scale).  A group that
 * holds an infinity or a NaN is kept as NaN.  No counterpart in the reference.
 *
 * codes, 1 byte an element, dense in x's layout class: (batch, dim, seqlen) for a channel-first x,
 * (batch, seqlen, dim) for a channel-last one; 16-byte aligned.  scales, 1 byte a group (the
 * exponent, biased by 127; 255: NaN), dense: (batch, dim, ceil(seqlen / 32)) or (batch, seqlen,
 * ceil(dim / 32)).
 */
#ifndef CC1D_CHECKPOINT_H_
#define CC1D_CHECKPOINT_H_

#include "cc1d.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cc1d_codes {
    uint8_t *codes;
    uint8_t *scales;
} cc1d_codes;

/* x -> codes, and codes -> x (a 16-bit float x is at most 65504).  Sizes, layout class and strides are
 * those of the x of a cc1d_fwd_params; its other fields are not read. */
int cc1d_checkpoint_e4m3(const cc1d_fwd_params *p, const cc1d_codes *to, cc1d_stream_t stream);
int cc1d_restore_e4m3(const cc1d_fwd_params *p, void *x, const cc1d_codes *from, cc1d_stream_t stream);

/* cc1d_fwd, and x kept: in one pass over x where it is channel-last, or channel-first in 16 bits with rows 32-byte
 * aligned and a multiple of 16 long, else by a second kernel. */
int cc1d_fwd_e4m3(const cc1d_fwd_params *p, const cc1d_codes *to, cc1d_stream_t stream);

/* cc1d_bwd with x taken from codes.  p->x itself is not read and may be NULL; x's strides say its
 * layout class.  `restored`: scratch of cc1d_bwd_e4m3_restore_bytes() bytes, 32-byte aligned; that is 0 where
 * the backward reads the codes as they are (16-bit types: channel-first rows as above, channel-last ones of a multiple of
 * 16 channels beside a channel-last dout), else room for a dense x. */
size_t cc1d_bwd_e4m3_restore_bytes(const cc1d_bwd_params *p);
int cc1d_bwd_e4m3(const cc1d_bwd_params *p, const cc1d_codes *from, void *restored, cc1d_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* CC1D_CHECKPOINT_H_ */
