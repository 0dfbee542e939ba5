/* Takes the place of the HIP runtime's launches: prints each one's grid and workgroup, and launches nothing. */
#include <stddef.h>
#include <stdio.h>

typedef struct { unsigned x, y, z; } dim3;
static dim3 grid, block;
static size_t lds;
static void* stream;

int __hipPushCallConfiguration(dim3 g, dim3 b, size_t l, void* s)
{
    grid = g, block = b, lds = l, stream = s;
    return 0;
}
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* l, void** s)
{
    *g = grid, *b = block, *l = lds, *s = stream;
    return 0;
}
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t l, void* s)
{
    (void)f, (void)args, (void)l, (void)s;
    printf("launch %u %u %u %u\n", g.x, g.y, g.z, b.x);
    fflush(stdout);
    return 0;
}
int hipGetLastError(void) { return 0; }
