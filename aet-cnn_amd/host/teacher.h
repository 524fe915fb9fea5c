/* teacher.h -- what the input pipeline (host/feeder.c) tells a network that
 * trains from a teacher (host/network.c); not part of the C-ABI headers. */
#ifndef AETCNN_TEACHER_H
#define AETCNN_TEACHER_H
#include "aetcnn_net.h"

/* The network's input are other images now: answers that a training forward
 * has read are those of earlier ones, and are forgotten. */
void an_images_fed(an_network *net);

#endif
